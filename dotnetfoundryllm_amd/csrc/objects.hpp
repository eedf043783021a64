// objects.hpp — the ABI's device context and buffers and its error reporting, shared by the files
// that define entry points of include/fllm.h.
#pragma once

#include "common.hpp"
#include "staging.hpp"

namespace fllm {

// Records the message that fllm_last_error returns and gives `code` back (api.hip).
int32_t fail(int32_t code, const char* fmt, ...);

#define HIP_TRY(expr)                                                                          \
    do {                                                                                       \
        hipError_t _e = (expr);                                                                \
        if (_e != hipSuccess) return fail(FLLM_E_DEVICE, "%s: %s", #expr, hipGetErrorString(_e)); \
    } while (0)

#define NOT_NULL(p)                                                  \
    do {                                                             \
        if (!(p)) return fail(FLLM_E_NULL, "%s must not be null", #p); \
    } while (0)

static const uint64_t kPad = 256;  // slack after every weight allocation for aligned over-reads

// Device memory that the calls on one context's stream share: `part` holds a call's partial results, dead
// once the call's last kernel has run; `cnt` counters that are zero between calls. Both grow and never
// shrink. A call holds `mu` while it enqueues, so that two threads' calls follow each other on the stream.
struct Workspace {
    std::mutex mu;
    uint8_t* part = nullptr;
    uint64_t part_bytes = 0;
    unsigned* cnt = nullptr;
    uint64_t n_cnt = 0;
};

// A batch's arrays on the device and the pinned block that they are copied from; `sent` says when the last copy has
// read it. Those of destroyed batches serve the next ones: calls still under way read `dev` before the stream's
// next copy into it.
struct BatchBlock {
    uint8_t *dev = nullptr, *pin = nullptr;
    uint64_t cap = 0;
    hipEvent_t sent = nullptr;
    bool in_flight = false;
};
struct SpareBlocks {
    static constexpr size_t kMost = 8;
    std::mutex mu;
    BatchBlock blocks[kMost];
    size_t n = 0;
};

}  // namespace fllm

struct fllm_ctx {
    int device = 0;
    hipStream_t stream = nullptr;
    int n_cu = 0;
    int64_t hbm = 0;
    fllm::Staging stage;
    uint8_t* scratch = nullptr;  // this device's address of the no-allocation scratch array
    hipError_t scratch_err = hipSuccess;  // why it could not be resolved, if so
    fllm::Workspace ws;          // partial results of the paged attention and of the draft check
    fllm::SpareBlocks spare;
};

struct fllm_buf {
    fllm_ctx* ctx = nullptr;
    uint8_t* ptr = nullptr;
    uint64_t n = 0;
    bool owned = true;  // false: the caller's memory (fllm_buf_wrap)
};
