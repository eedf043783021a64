// pages_attend_q4_0.hip — attention over Q4_0 pages.
#include "pages_attend.hpp"

namespace fllm {

hipError_t launch_attend_q4_0(const PagesView& pg, const BatchView& b, const AttnWork& w, const RowsView& q, const RowsView& out,
                            float scale, float softcap, hipStream_t st) {
    return launch_items_of<FLLM_TYPE_Q4_0>(attend_args(pg, b, w, q, out, scale, softcap), w, st);
}

}  // namespace fllm
