// pages.hpp — launch interface of the paged K/V cache kernels: rows into and out of the pages
// (pages.hip), attention over them (pages_attention.hip), and the check of drafted tokens (draft.hip).
#pragma once

#include "common.hpp"
#include "pages_plan.hpp"

namespace fllm {

// One layer's pages: cell (page, kv head) of K at k + (page * nkv + head) * cell, its codes, then at
// scale_off its scales (layouts in fllm.h).
struct PagesView {
    uint8_t *k, *v;
    int type, nkv, hd, page_log2;
    uint64_t cell;
    uint32_t scale_off;
};
// A batch on the device: per sequence {first row of its new tokens, their number, its length, first row of its
// positions} and where its pages start in `tables`; the pages with new tokens (PageTile).
struct BatchView {
    const int4* seqs;
    const int* first;
    const int* tables;
    const int4* new_tiles;
    int n_seqs, n_new_tiles, n_blocks;  // n_blocks: pages of all sequences
    int n_rows, max_new;                // new tokens of all sequences, most of one
    int n_heads, window;
};
struct RowsView {
    uint8_t* p;
    int64_t ld;
    int type;
};

// the new rows into their pages / rows out of the pages (k.p or v.p null: not read)
hipError_t launch_pages_append(const PagesView& pg, const BatchView& b, const RowsView& k, const RowsView& v, hipStream_t st);
hipError_t launch_pages_read(const PagesView& pg, const BatchView& b, bool new_only, const RowsView& k, const RowsView& v,
                             hipStream_t st);
// Attention items on the device (pages_plan.hpp), a list for each class of tiles; part: room
// for part_rows * nkv rows of head_dim floats, then a max and a sum for each; cnt: as many zeros, left as zeros.
struct AttnWork {
    const AttnItem* items[kAttnClasses];
    int n[kAttnClasses];
    float* part;
    unsigned* cnt;
    int64_t part_rows;
    // steps that are turned into images first: room for images * nkv * 64 keys of K and V (attend_image_bytes) and for
    // 4 floats each
    const ImageItem* image_items;
    int n_image_items;
    int64_t n_images;
    void* images;
    float* image_units;
};
hipError_t launch_pages_attention(const PagesView& pg, const BatchView& b, const AttnWork& w, const RowsView& q,
                                  const RowsView& out, float scale, float softcap, hipStream_t st);

// the same for one cache type each
hipError_t launch_attend_f16(const PagesView& pg, const BatchView& b, const AttnWork& w, const RowsView& q, const RowsView& out,
                             float scale, float softcap, hipStream_t st);
hipError_t launch_attend_q8_0(const PagesView& pg, const BatchView& b, const AttnWork& w, const RowsView& q, const RowsView& out,
                              float scale, float softcap, hipStream_t st);
hipError_t launch_attend_q4_0(const PagesView& pg, const BatchView& b, const AttnWork& w, const RowsView& q, const RowsView& out,
                              float scale, float softcap, hipStream_t st);

struct DraftView {
    int n_seqs, n_draft, vocab;
    const float* target;
    int64_t target_ld;
    const float* draft;  // null: one-point distributions
    int64_t draft_ld;
    const int *tokens, *counts;  // counts null: n_draft
    const float *u_accept, *u_sample;
    int *out_tokens, *out_counts;
};
// A row's segments of *seg ids each, a workgroup per sequence and segment; vocab up to kDraftVocab.
constexpr int kDraftVocab = 1 << 20;
int draft_segments(int n_seqs, int vocab, int n_cu, int* seg, int* runs);
// part: 2 doubles per sequence and segment; cnt: a zero per sequence, left as one
hipError_t launch_draft_verify(const DraftView& d, int seg, int n_seg, int runs, double* part, unsigned* cnt, hipStream_t st);

// ---- elements ---------------------------------------------------------------------------
// round to nearest even; a NaN stays one
__device__ __forceinline__ uint16_t bf16_round(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

}  // namespace fllm
