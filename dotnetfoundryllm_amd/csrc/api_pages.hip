// api_pages.hip — the paged K/V cache and the draft check in the C ABI (include/fllm.h): descriptions,
// batches and argument checks; the kernels are in pages.hip, pages_attention.hip and draft.hip.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <mutex>
#include <new>
#include <vector>

#include "objects.hpp"
#include "pages.hpp"
#include "pages_plan.hpp"

using namespace fllm;

struct fllm_pages {
    fllm_ctx* ctx = nullptr;
    fllm_pages_desc d{};
    uint8_t* ptr = nullptr;
    bool owned = false;
    uint64_t cell = 0;
    int n_batches = 0;
    bool disposed = false;
};

struct fllm_batch {
    fllm_pages* p = nullptr;
    int n_heads = 0, window = 0;
    BatchPlan plan;
    AttnPlan attn;
    BatchBlock mem;
    BatchView view{};
    AttnWork work{};
};

// Runs a body that may allocate on the host: no exception crosses the ABI.
template <typename F>
static int32_t guarded(F body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return fail(FLLM_E_OOM, "out of host memory");
    } catch (...) {
        return fail(FLLM_E_INVALID_OP, "unexpected exception");
    }
}

// =====================================================================================
// pages
// =====================================================================================
extern "C" int32_t fllm_pages_bytes(const fllm_pages_desc* desc, uint64_t* out) {
    NOT_NULL(desc);
    NOT_NULL(out);
    BatchError e;
    if (pages_desc_check(*desc, out, &e)) return fail(e.code, "%s", e.text);
    return FLLM_OK;
}

extern "C" int32_t fllm_pages_create(fllm_ctx* ctx, const fllm_pages_desc* desc, fllm_buf* mem, uint64_t offset,
                                     fllm_pages** out) {
    NOT_NULL(ctx);
    NOT_NULL(desc);
    NOT_NULL(out);
    *out = nullptr;
    uint64_t bytes = 0;
    BatchError err;
    if (pages_desc_check(*desc, &bytes, &err)) return fail(err.code, "%s", err.text);
    if (mem) {
        if (mem->ctx != ctx) return fail(FLLM_E_ARG, "the buffer belongs to another context");
        if (offset % 16 != 0) return fail(FLLM_E_ARG, "offset must be a multiple of 16");
        if (offset > mem->n || bytes > mem->n - offset)
            return fail(FLLM_E_ARG, "the pages take %llu bytes at %llu of a buffer of %llu", (unsigned long long)bytes,
                        (unsigned long long)offset, (unsigned long long)mem->n);
    }
    fllm_pages* p = new (std::nothrow) fllm_pages();
    if (!p) return fail(FLLM_E_OOM, "out of host memory");
    p->ctx = ctx;
    p->d = *desc;
    p->cell = pages_cell_bytes(*desc);
    if (mem) {
        p->ptr = mem->ptr + offset;
    } else {
        hipError_t e = hipSetDevice(ctx->device);
        if (e == hipSuccess) e = hipMalloc(&p->ptr, bytes);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            delete p;
            return fail(e == hipErrorOutOfMemory ? FLLM_E_OOM : FLLM_E_DEVICE, "hipMalloc(%llu): %s", (unsigned long long)bytes,
                        hipGetErrorString(e));
        }
        p->owned = true;
        e = hipMemsetAsync(p->ptr, 0, bytes, ctx->stream);
        if (e != hipSuccess) {
            hipFree(p->ptr);
            delete p;
            return fail(FLLM_E_DEVICE, "hipMemsetAsync: %s", hipGetErrorString(e));
        }
    }
    *out = p;
    return FLLM_OK;
}

static void pages_free(fllm_pages* p) {
    hipSetDevice(p->ctx->device);
    hipStreamSynchronize(p->ctx->stream);
    if (p->owned) hipFree(p->ptr);
    delete p;
}

extern "C" int32_t fllm_pages_destroy(fllm_pages* p) {
    if (!p) return FLLM_OK;
    p->disposed = true;
    if (p->n_batches == 0) pages_free(p);
    return FLLM_OK;
}

// =====================================================================================
// batches
// =====================================================================================
extern "C" int32_t fllm_batch_create(fllm_pages* p, int32_t n_heads, int32_t window, fllm_batch** out) {
    NOT_NULL(p);
    NOT_NULL(out);
    *out = nullptr;
    if (p->disposed) return fail(FLLM_E_DISPOSED, "the pages were destroyed");
    if (n_heads < 1 || n_heads > 65535 || n_heads % p->d.n_kv_heads != 0)
        return fail(FLLM_E_ARG, "%d query heads over %d kv heads", n_heads, p->d.n_kv_heads);
    if (window < 1) return fail(FLLM_E_ARG_RANGE, "window must be positive");
    HIP_TRY(hipSetDevice(p->ctx->device));
    return guarded([&]() -> int32_t {
        fllm_batch* b = new fllm_batch();
        SpareBlocks& spare = p->ctx->spare;
        {
            std::lock_guard<std::mutex> lock(spare.mu);
            if (spare.n) b->mem = spare.blocks[--spare.n];
        }
        const hipError_t e = b->mem.sent ? hipSuccess : hipEventCreateWithFlags(&b->mem.sent, hipEventDisableTiming);
        if (e != hipSuccess) {
            delete b;
            return fail(FLLM_E_DEVICE, "hipEventCreate: %s", hipGetErrorString(e));
        }
        b->p = p;
        b->n_heads = n_heads;
        b->window = window;
        p->n_batches++;
        *out = b;
        return FLLM_OK;
    });
}

// Room for n bytes on the device and in the pinned block. The old memory may still be read by enqueued
// calls: they are waited for first.
static hipError_t batch_room(fllm_ctx* ctx, BatchBlock* b, uint64_t n) {
    hipError_t e = hipSuccess;
    if (b->in_flight) e = hipEventSynchronize(b->sent);
    b->in_flight = false;
    if (e != hipSuccess || n <= b->cap) return e;
    e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) return e;
    if (b->dev) hipFree(b->dev);
    if (b->pin) hipHostFree(b->pin);
    b->dev = b->pin = nullptr;
    b->cap = 0;
    const uint64_t want = n + n / 2 + 4096;
    e = hipMalloc(&b->dev, want);
    if (e == hipSuccess) e = hipHostMalloc((void**)&b->pin, want, hipHostMallocDefault);
    if (e == hipSuccess) b->cap = want;
    else (void)hipGetLastError();  // reported here: not to be found by the next launch
    return e;
}

extern "C" int32_t fllm_batch_set(fllm_batch* b, int32_t n_seqs, const int32_t* new_tokens, const int32_t* lengths,
                                  const int32_t* tables, int64_t ld) {
    NOT_NULL(b);
    fllm_pages* p = b->p;
    b->view = BatchView{};
    b->work = AttnWork{};
    if (p->disposed) return fail(FLLM_E_DISPOSED, "the pages were destroyed");
    if (n_seqs < 0) return fail(FLLM_E_ARG_RANGE, "n_seqs must not be negative");
    if (n_seqs == 0) {
        b->plan = BatchPlan{};
        return FLLM_OK;
    }
    NOT_NULL(new_tokens);
    NOT_NULL(lengths);
    NOT_NULL(tables);
    if (ld < 0) return fail(FLLM_E_ARG_RANGE, "ld must not be negative");
    HIP_TRY(hipSetDevice(p->ctx->device));
    return guarded([&]() -> int32_t {
        BatchError err;
        if (batch_plan(p->d, b->window, n_seqs, new_tokens, lengths, tables, ld, &b->plan, &err)) {
            b->plan.n_seqs = b->plan.n_rows = b->plan.n_pos = 0;
            return fail(err.code, "%s", err.text);
        }
        const BatchPlan& pl = b->plan;
        const int n_plan_seqs = pl.n_seqs;
        if (!attn_plan(pl, b->n_heads, p->d.n_kv_heads, p->d.head_dim, p->d.type != FLLM_TYPE_F16, b->window, p->ctx->n_cu, &b->attn)) {
            b->plan.n_seqs = b->plan.n_rows = b->plan.n_pos = 0;
            return fail(FLLM_E_ARG, "the batch is too large");
        }
        b->plan.n_seqs = 0;  // empty until everything is on its way
        // sequences, items, images, tiles, starts, tables: parts of 16, 64, 32, 16 and 4 bytes
        constexpr int N = kAttnClasses + 5;
        const void* from[N] = {pl.seqs.data()};
        uint64_t size[N] = {(pl.seqs.size() * sizeof(SeqPlan) + 63) / 64 * 64}, at[N + 1] = {0};
        const auto part = [&](int i, const auto& v) { from[i] = v.data(), size[i] = v.size() * sizeof(v[0]); };
        for (int i = 0; i < kAttnClasses; i++) part(1 + i, b->attn.items[i]);
        part(N - 4, b->attn.image_items);
        part(N - 3, pl.new_tiles);
        part(N - 2, pl.first);
        part(N - 1, pl.tables);
        for (int i = 0; i < N; i++) at[i + 1] = at[i] + size[i];
        hipError_t e = batch_room(p->ctx, &b->mem, at[N]);
        if (e != hipSuccess)
            return fail(e == hipErrorOutOfMemory ? FLLM_E_OOM : FLLM_E_DEVICE, "batch memory: %s", hipGetErrorString(e));
        for (int i = 0; i < N; i++)
            if (size[i]) memcpy(b->mem.pin + at[i], from[i], i ? size[i] : pl.seqs.size() * sizeof(SeqPlan));
        HIP_TRY(hipMemcpyAsync(b->mem.dev, b->mem.pin, at[N], hipMemcpyHostToDevice, p->ctx->stream));
        HIP_TRY(hipEventRecord(b->mem.sent, p->ctx->stream));
        b->mem.in_flight = true;
        b->plan.n_seqs = n_plan_seqs;
        b->view.seqs = (const int4*)b->mem.dev;
        b->view.tables = (const int*)(b->mem.dev + at[N - 1]);
        b->view.first = (const int*)(b->mem.dev + at[N - 2]);
        b->view.new_tiles = (const int4*)(b->mem.dev + at[N - 3]);
        b->view.n_seqs = n_plan_seqs;
        b->view.n_new_tiles = (int)pl.new_tiles.size();
        b->view.n_blocks = (int)pl.tables.size();
        b->view.n_rows = pl.n_rows;
        b->view.max_new = pl.max_new;
        b->view.n_heads = b->n_heads;
        b->view.window = b->window;
        for (int i = 0; i < kAttnClasses; i++) {
            b->work.items[i] = (const AttnItem*)(b->mem.dev + at[1 + i]);
            b->work.n[i] = (int)b->attn.items[i].size();
        }
        b->work.part_rows = b->attn.part_rows;
        b->work.image_items = (const ImageItem*)(b->mem.dev + at[N - 4]);
        b->work.n_image_items = (int)b->attn.image_items.size();
        b->work.n_images = b->attn.images;
        return FLLM_OK;
    });
}

extern "C" int32_t fllm_batch_destroy(fllm_batch* b) {
    if (!b) return FLLM_OK;
    fllm_pages* p = b->p;
    SpareBlocks& spare = p->ctx->spare;
    bool kept = false;
    {
        std::lock_guard<std::mutex> lock(spare.mu);
        if (spare.n < SpareBlocks::kMost) spare.blocks[spare.n++] = b->mem, kept = true;
    }
    if (!kept) {
        hipSetDevice(p->ctx->device);
        hipStreamSynchronize(p->ctx->stream);
        if (b->mem.dev) hipFree(b->mem.dev);
        if (b->mem.pin) hipHostFree(b->mem.pin);
        hipEventDestroy(b->mem.sent);
    }
    delete b;
    p->n_batches--;
    if (p->disposed && p->n_batches == 0) pages_free(p);
    return FLLM_OK;
}

// =====================================================================================
// calls
// =====================================================================================
// Room in the context's workspace (its mutex is held). Memory that earlier calls use is waited for
// before it is replaced.
static hipError_t workspace_room(fllm_ctx* ctx, uint64_t part_bytes, uint64_t n_cnt) {
    Workspace& w = ctx->ws;
    if (part_bytes <= w.part_bytes && n_cnt <= w.n_cnt) return hipSuccess;
    hipError_t e = hipStreamSynchronize(ctx->stream);
    if (e == hipSuccess && part_bytes > w.part_bytes) {
        if (w.part) hipFree(w.part);
        w.part = nullptr;
        w.part_bytes = 0;
        const uint64_t want = part_bytes + std::min<uint64_t>(part_bytes / 2, (uint64_t)64 << 20);
        e = hipMalloc(&w.part, want);
        if (e == hipSuccess) w.part_bytes = want;
    }
    if (e == hipSuccess && n_cnt > w.n_cnt) {
        if (w.cnt) hipFree(w.cnt);
        w.cnt = nullptr;
        w.n_cnt = 0;
        const uint64_t n = n_cnt + n_cnt / 2;
        e = hipMalloc(&w.cnt, n * sizeof(unsigned));
        if (e == hipSuccess) e = hipMemsetAsync(w.cnt, 0, n * sizeof(unsigned), ctx->stream);
        if (e == hipSuccess) w.n_cnt = n;
    }
    if (e != hipSuccess) (void)hipGetLastError();
    return e;
}

// Rows that a call reads or writes: `n` of them, `width` elements wide, each aligned to `align` bytes.
static int32_t check_rows(fllm_ctx* ctx, const fllm_rows* r, const char* name, int64_t n, int64_t width, RowsView* out,
                          uint64_t align = 16) {
    if (!r || !r->buf) return fail(FLLM_E_NULL, "%s must not be null", name);
    if (r->buf->ctx != ctx) return fail(FLLM_E_ARG, "%s: the buffer belongs to another context", name);
    if (r->type != FLLM_TYPE_F32 && r->type != FLLM_TYPE_F16 && r->type != FLLM_TYPE_BF16)
        return fail(FLLM_E_NOT_SUPPORTED, "%s: rows of type %d are not supported", name, r->type);
    const uint64_t esz = r->type == FLLM_TYPE_F32 ? 4 : 2;
    if (r->ld < width || r->ld > INT64_MAX / 8 || (uint64_t)r->ld * esz % align != 0 || r->offset % align != 0)
        return fail(FLLM_E_ARG, "%s: offset %llu, ld %lld for rows of %lld elements (both multiples of %llu bytes)", name,
                    (unsigned long long)r->offset, (long long)r->ld, (long long)width, (unsigned long long)align);
    if (n > 0) {
        const unsigned __int128 end = (unsigned __int128)r->offset + ((unsigned __int128)(n - 1) * (uint64_t)r->ld + (uint64_t)width) * esz;
        if (end > r->buf->n)
            return fail(FLLM_E_ARG, "%s: %lld rows do not fit a buffer of %llu bytes", name, (long long)n, (unsigned long long)r->buf->n);
    }
    out->p = r->buf->ptr + r->offset;
    out->ld = r->ld;
    out->type = r->type;
    return FLLM_OK;
}

// Whether n rows of each share memory: exact for rows of one stride (columns of one matrix), else by their ranges.
static bool overlap(const RowsView& a, const RowsView& b, int64_t n, int64_t width) {
    if (n <= 0) return false;
    const auto size = [](const RowsView& r) { return (int64_t)(r.type == FLLM_TYPE_F32 ? 4 : 2); };
    const auto end = [&](const RowsView& r) { return r.p + ((n - 1) * r.ld + width) * size(r); };
    if (!(a.p < end(b) && b.p < end(a))) return false;
    const int64_t stride = a.ld * size(a);
    if (stride != b.ld * size(b)) return true;
    const int64_t d = b.p - a.p, first = -d / stride;
    for (int64_t k = first - 1; k <= first + 1; k++)  // row i of a and row i + k of b
        if (k > -n && k < n && d + k * stride < width * size(a) && d + k * stride > -width * size(b)) return true;
    return false;
}

// Rows of a call on pages must not lie in the pages themselves.
static int32_t check_apart(const fllm_pages* p, const RowsView& r, const char* name, int64_t n, int64_t width) {
    if (n <= 0) return FLLM_OK;
    const uint8_t* end = r.p + ((n - 1) * r.ld + width) * (r.type == FLLM_TYPE_F32 ? 4 : 2);
    const uint64_t bytes = 2 * p->cell * (uint64_t)p->d.n_kv_heads * (uint64_t)p->d.n_pages * (uint64_t)p->d.n_layers;
    return r.p < p->ptr + bytes && p->ptr < end ? fail(FLLM_E_ARG, "%s overlaps the pages", name) : FLLM_OK;
}

static int32_t check_call(fllm_batch* b, int32_t layer) {
    NOT_NULL(b);
    if (b->p->disposed) return fail(FLLM_E_DISPOSED, "the pages were destroyed");
    if (layer < 0 || layer >= b->p->d.n_layers)
        return fail(FLLM_E_ARG_RANGE, "Layer index must be in [0, %d].", b->p->d.n_layers - 1);
    return FLLM_OK;
}

static PagesView pages_view(const fllm_pages* p, int layer) {
    const uint64_t half = p->cell * (uint64_t)p->d.n_kv_heads * (uint64_t)p->d.n_pages;
    PagesView v{};
    v.k = p->ptr + 2 * half * (uint64_t)layer;
    v.v = v.k + half;
    v.type = p->d.type;
    v.nkv = p->d.n_kv_heads;
    v.hd = p->d.head_dim;
    v.page_log2 = p->d.page_size == 16 ? 4 : p->d.page_size == 32 ? 5 : p->d.page_size == 64 ? 6 : 7;
    v.cell = p->cell;
    v.scale_off = (uint32_t)pages_code_bytes(p->d);
    return v;
}

extern "C" int32_t fllm_pages_append(fllm_batch* b, int32_t layer, const fllm_rows* k, const fllm_rows* v) {
    int32_t rc = check_call(b, layer);
    if (rc) return rc;
    fllm_pages* p = b->p;
    const int64_t width = (int64_t)p->d.n_kv_heads * p->d.head_dim;
    RowsView rk{}, rv{};
    if ((rc = check_rows(p->ctx, k, "k", b->view.n_rows, width, &rk))) return rc;
    if ((rc = check_rows(p->ctx, v, "v", b->view.n_rows, width, &rv))) return rc;
    if ((rc = check_apart(p, rk, "k", b->view.n_rows, width)) || (rc = check_apart(p, rv, "v", b->view.n_rows, width))) return rc;
    if (b->view.n_rows == 0) return FLLM_OK;
    HIP_TRY(hipSetDevice(p->ctx->device));
    HIP_TRY(launch_pages_append(pages_view(p, layer), b->view, rk, rv, p->ctx->stream));
    return FLLM_OK;
}

extern "C" int32_t fllm_pages_read(fllm_batch* b, int32_t layer, int32_t new_only, const fllm_rows* k, const fllm_rows* v) {
    int32_t rc = check_call(b, layer);
    if (rc) return rc;
    if (new_only != 0 && new_only != 1) return fail(FLLM_E_ARG_RANGE, "new_only must be 0 or 1");
    fllm_pages* p = b->p;
    const int64_t width = (int64_t)p->d.n_kv_heads * p->d.head_dim;
    const int64_t n = b->view.n_seqs == 0 ? 0 : new_only ? b->view.n_rows : b->plan.n_pos;
    RowsView rk{}, rv{};
    if (!k && !v) return fail(FLLM_E_NULL, "k and v must not both be null");
    if (k && (rc = check_rows(p->ctx, k, "k", n, width, &rk))) return rc;
    if (v && (rc = check_rows(p->ctx, v, "v", n, width, &rv))) return rc;
    if ((k && (rc = check_apart(p, rk, "k", n, width))) || (v && (rc = check_apart(p, rv, "v", n, width)))) return rc;
    if (k && v && overlap(rk, rv, n, width)) return fail(FLLM_E_ARG, "k and v overlap");
    if (!new_only && b->view.n_seqs && b->plan.holes) return fail(FLLM_E_INVALID_OP, "pages before the window were given back");
    if (n == 0) return FLLM_OK;
    HIP_TRY(hipSetDevice(p->ctx->device));
    HIP_TRY(launch_pages_read(pages_view(p, layer), b->view, new_only != 0, rk, rv, p->ctx->stream));
    return FLLM_OK;
}

extern "C" int32_t fllm_pages_attention(fllm_batch* b, int32_t layer, const fllm_rows* q, const fllm_rows* out, float scale,
                                        float softcap) {
    int32_t rc = check_call(b, layer);
    if (rc) return rc;
    fllm_pages* p = b->p;
    const int64_t width = (int64_t)b->n_heads * p->d.head_dim;
    RowsView rq{}, ro{};
    if ((rc = check_rows(p->ctx, q, "q", b->view.n_rows, width, &rq))) return rc;
    if ((rc = check_rows(p->ctx, out, "out", b->view.n_rows, width, &ro))) return rc;
    if ((rc = check_apart(p, rq, "q", b->view.n_rows, width)) || (rc = check_apart(p, ro, "out", b->view.n_rows, width))) return rc;
    if (overlap(rq, ro, b->view.n_rows, width)) return fail(FLLM_E_ARG, "q and out overlap");
    if (!isfinite(scale)) return fail(FLLM_E_ARG_RANGE, "scale must be finite");
    if (!isfinite(softcap) || softcap < 0.0f) return fail(FLLM_E_ARG_RANGE, "softcap must be finite and not negative");
    if (b->view.n_rows == 0) return FLLM_OK;
    HIP_TRY(hipSetDevice(p->ctx->device));
    std::lock_guard<std::mutex> lock(p->ctx->ws.mu);
    AttnWork w = b->work;
    const uint64_t rows = (uint64_t)w.part_rows * (uint64_t)p->d.n_kv_heads;
    const uint64_t part = (rows * (uint64_t)(p->d.head_dim + 2) * sizeof(float) + 255) / 256 * 256;
    const uint64_t images = (uint64_t)w.n_images * (uint64_t)p->d.n_kv_heads;
    const uint64_t image = images * attend_image_bytes(p->d.head_dim, rq.type == FLLM_TYPE_F32 || ro.type == FLLM_TYPE_F32);
    hipError_t e = workspace_room(p->ctx, part + image + images * 4 * sizeof(float), rows);
    if (e != hipSuccess)
        return fail(e == hipErrorOutOfMemory ? FLLM_E_OOM : FLLM_E_DEVICE, "attention workspace: %s", hipGetErrorString(e));
    w.part = (float*)p->ctx->ws.part;
    w.cnt = p->ctx->ws.cnt;
    w.images = p->ctx->ws.part + part;
    w.image_units = (float*)(p->ctx->ws.part + part + image);
    HIP_TRY(launch_pages_attention(pages_view(p, layer), b->view, w, rq, ro, scale, softcap, p->ctx->stream));
    return FLLM_OK;
}

// =====================================================================================
// drafted tokens
// =====================================================================================
// n 4-byte values in a buffer of the context.
static int32_t check_values(fllm_ctx* ctx, const fllm_buf* b, const char* name, int64_t n) {
    if (!b) return fail(FLLM_E_NULL, "%s must not be null", name);
    if (b->ctx != ctx) return fail(FLLM_E_ARG, "%s: the buffer belongs to another context", name);
    if ((uint64_t)n > b->n / 4) return fail(FLLM_E_ARG, "%s: %lld values do not fit a buffer of %llu bytes", name, (long long)n, (unsigned long long)b->n);
    return FLLM_OK;
}

extern "C" int32_t fllm_draft_verify(fllm_ctx* ctx, const fllm_draft_desc* d) {
    NOT_NULL(ctx);
    NOT_NULL(d);
    if (d->n_seqs < 0 || d->n_draft < 0 || d->vocab < 1)
        return fail(FLLM_E_ARG_RANGE, "%d sequences, %d drafted tokens, vocabulary %d", d->n_seqs, d->n_draft, d->vocab);
    if (d->vocab > kDraftVocab) return fail(FLLM_E_NOT_SUPPORTED, "vocabularies above %d are not supported", kDraftVocab);
    const int64_t n = d->n_seqs, nd = n * d->n_draft, nt = n * ((int64_t)d->n_draft + 1);
    RowsView target{}, draft{};
    int32_t rc;
    if ((rc = check_rows(ctx, &d->target, "target", nt, d->vocab, &target, 4))) return rc;
    if (d->draft.buf && (rc = check_rows(ctx, &d->draft, "draft", nd, d->vocab, &draft, 4))) return rc;
    if (target.type != FLLM_TYPE_F32 || (d->draft.buf && draft.type != FLLM_TYPE_F32))
        return fail(FLLM_E_NOT_SUPPORTED, "probabilities are F32");
    if (d->n_draft) {
        if ((rc = check_values(ctx, d->tokens, "tokens", nd))) return rc;
        if ((rc = check_values(ctx, d->u_accept, "u_accept", nd))) return rc;
    }
    if (d->counts && (rc = check_values(ctx, d->counts, "counts", n))) return rc;
    if ((rc = check_values(ctx, d->u_sample, "u_sample", n))) return rc;
    if ((rc = check_values(ctx, d->out_tokens, "out_tokens", nt))) return rc;
    if ((rc = check_values(ctx, d->out_counts, "out_counts", n))) return rc;
    if (n == 0) return FLLM_OK;
    // the outputs are written while other sequences' inputs are still read
    const uint8_t* outs[2] = {d->out_tokens->ptr, d->out_counts->ptr};
    const uint64_t out_bytes[2] = {4 * (uint64_t)nt, 4 * (uint64_t)n};
    const auto meet = [&](const uint8_t* p, uint64_t bytes, int o) { return p && bytes && p < outs[o] + out_bytes[o] && outs[o] < p + bytes; };
    const auto rows_bytes = [&](const RowsView& r, int64_t m) { return m ? (uint64_t)((m - 1) * r.ld + d->vocab) * 4 : 0; };
    for (int o = 0; o < 2; o++) {
        const bool bad = meet(target.p, rows_bytes(target, nt), o) || meet(draft.p, rows_bytes(draft, nd), o) ||
                         (d->n_draft && (meet(d->tokens->ptr, 4 * (uint64_t)nd, o) || meet(d->u_accept->ptr, 4 * (uint64_t)nd, o))) ||
                         (d->counts && meet(d->counts->ptr, 4 * (uint64_t)n, o)) || meet(d->u_sample->ptr, 4 * (uint64_t)n, o) ||
                         (o == 0 && meet(outs[1], out_bytes[1], 0));
        if (bad) return fail(FLLM_E_ARG, "%s overlaps another argument", o ? "out_counts" : "out_tokens");
    }
    HIP_TRY(hipSetDevice(ctx->device));
    DraftView v{};
    v.n_seqs = d->n_seqs;
    v.n_draft = d->n_draft;
    v.vocab = d->vocab;
    v.target = (const float*)target.p;
    v.target_ld = target.ld;
    v.draft = (const float*)draft.p;
    v.draft_ld = draft.ld;
    v.tokens = d->n_draft ? (const int*)d->tokens->ptr : nullptr;
    v.counts = d->counts ? (const int*)d->counts->ptr : nullptr;
    v.u_accept = d->n_draft ? (const float*)d->u_accept->ptr : nullptr;
    v.u_sample = (const float*)d->u_sample->ptr;
    v.out_tokens = (int*)d->out_tokens->ptr;
    v.out_counts = (int*)d->out_counts->ptr;
    int seg = 0, runs = 1;
    const int n_seg = draft_segments(v.n_seqs, v.vocab, ctx->n_cu, &seg, &runs);
    std::lock_guard<std::mutex> lock(ctx->ws.mu);
    hipError_t e = workspace_room(ctx, (uint64_t)n * (uint64_t)n_seg * 16, (uint64_t)n);
    if (e != hipSuccess)
        return fail(e == hipErrorOutOfMemory ? FLLM_E_OOM : FLLM_E_DEVICE, "draft workspace: %s", hipGetErrorString(e));
    HIP_TRY(launch_draft_verify(v, seg, n_seg, runs, (double*)ctx->ws.part, ctx->ws.cnt, ctx->stream));
    return FLLM_OK;
}
