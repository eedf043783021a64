// pages_attention.hip — attention of new tokens over the pages of their sequences: the cache types' launches
// (pages_attend.hpp).
#include "pages.hpp"

namespace fllm {

hipError_t launch_pages_attention(const PagesView& pg, const BatchView& b, const AttnWork& w, const RowsView& q,
                                  const RowsView& out, float scale, float softcap, hipStream_t st) {
    switch (pg.type) {
        case FLLM_TYPE_F16: return launch_attend_f16(pg, b, w, q, out, scale, softcap, st);
        case FLLM_TYPE_Q8_0: return launch_attend_q8_0(pg, b, w, q, out, scale, softcap, st);
        case FLLM_TYPE_Q4_0: return launch_attend_q4_0(pg, b, w, q, out, scale, softcap, st);
    }
    return hipErrorNotSupported;
}

}  // namespace fllm
