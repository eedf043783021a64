// The batch planner of the paged K/V cache (csrc/pages_plan.hpp) behind a C interface, for
// tests/test_pages_plan.py.
#include <cstring>

#include "../dotnetfoundryllm_amd/csrc/pages_plan.hpp"

using namespace fllm;

static BatchPlan g_plan;
static AttnPlan g_attn;
static BatchError g_err;

extern "C" int32_t plan_set(const fllm_pages_desc* d, int32_t n_heads, int32_t window, int32_t n_cu, int32_t n_seqs,
                            const int32_t* n_new, const int32_t* lengths, const int32_t* tables, int64_t ld) {
    if (batch_plan(*d, window, n_seqs, n_new, lengths, tables, ld, &g_plan, &g_err)) return g_err.code;
    return attn_plan(g_plan, n_heads, d->n_kv_heads, d->head_dim, d->type != FLLM_TYPE_F16, window, n_cu, &g_attn) ? 0 : -100;
}
extern "C" const char* plan_error() { return g_err.text; }
extern "C" int64_t plan_items(int32_t c, AttnItem* out) {
    if (out && !g_attn.items[c].empty()) memcpy(out, g_attn.items[c].data(), g_attn.items[c].size() * sizeof(AttnItem));
    return (int64_t)g_attn.items[c].size();
}
extern "C" int64_t plan_images(ImageItem* out, int64_t* total) {
    if (out && !g_attn.image_items.empty()) memcpy(out, g_attn.image_items.data(), g_attn.image_items.size() * sizeof(ImageItem));
    *total = g_attn.images;
    return (int64_t)g_attn.image_items.size();
}
extern "C" int64_t plan_part_rows() { return g_attn.part_rows; }
extern "C" void plan_sizes(int32_t* out) {
    const int32_t v[] = {g_plan.n_seqs, g_plan.n_rows, g_plan.n_pos, (int32_t)g_plan.tables.size(),
                         (int32_t)g_plan.new_tiles.size(), (int32_t)g_plan.first.size(), g_plan.max_new, g_plan.holes};
    memcpy(out, v, sizeof(v));
}
extern "C" void plan_tables(int32_t* out) {
    if (!g_plan.tables.empty()) memcpy(out, g_plan.tables.data(), g_plan.tables.size() * 4);
}
extern "C" void plan_first(int32_t* out) { memcpy(out, g_plan.first.data(), g_plan.first.size() * 4); }
extern "C" void plan_tiles(PageTile* out) {
    if (!g_plan.new_tiles.empty()) memcpy(out, g_plan.new_tiles.data(), g_plan.new_tiles.size() * sizeof(PageTile));
}
extern "C" int32_t plan_desc(const fllm_pages_desc* d, uint64_t* bytes) { return pages_desc_check(*d, bytes, &g_err); }
