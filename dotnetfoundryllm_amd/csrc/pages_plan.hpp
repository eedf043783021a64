// pages_plan.hpp — what the host works out for a batch over the paged K/V cache: the checks of its
// lengths and page tables, and the attention's work items. Plain C++ without the HIP API, so the CPU
// tests compile it by itself.
#pragma once

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <vector>

#include "../../include/fllm.h"

namespace fllm {

constexpr int kPagesMaxLength = 1 << 30;  // positions of a sequence

// Bytes of one cell (a page of one kv head, K or V); 0 where the description is not a valid one.
inline uint64_t pages_cell_bytes(const fllm_pages_desc& d) {
    const uint64_t n = (uint64_t)d.page_size * (uint64_t)d.head_dim;
    switch (d.type) {
        case FLLM_TYPE_F16: return 2 * n;
        case FLLM_TYPE_Q8_0: return n / 32 * 34;
        case FLLM_TYPE_Q4_0: return n / 32 * 18;
    }
    return 0;
}

// Bytes of a cell's codes: its scales start there.
inline uint64_t pages_code_bytes(const fllm_pages_desc& d) {
    const uint64_t n = (uint64_t)d.page_size * (uint64_t)d.head_dim;
    return d.type == FLLM_TYPE_F16 ? 2 * n : d.type == FLLM_TYPE_Q8_0 ? n : n / 2;
}

struct BatchError {
    int32_t code = FLLM_OK;
    char text[200] = "";
};

inline int32_t pages_desc_check(const fllm_pages_desc& d, uint64_t* bytes, BatchError* e) {
    e->code = FLLM_E_ARG;
    if (d.type != FLLM_TYPE_F16 && d.type != FLLM_TYPE_Q8_0 && d.type != FLLM_TYPE_Q4_0) {
        snprintf(e->text, sizeof(e->text), "pages of type %d are not supported", d.type);
        return e->code = FLLM_E_NOT_SUPPORTED;
    }
    if (d.head_dim < 32 || d.head_dim > 256 || d.head_dim % 32 != 0) {
        snprintf(e->text, sizeof(e->text), "head_dim %d is not a multiple of 32 in [32, 256]", d.head_dim);
        return e->code;
    }
    if (d.page_size != 16 && d.page_size != 32 && d.page_size != 64 && d.page_size != 128) {
        snprintf(e->text, sizeof(e->text), "page_size %d is not 16, 32, 64 or 128", d.page_size);
        return e->code;
    }
    if (d.n_layers < 1 || d.n_kv_heads < 1 || d.n_kv_heads > 1024 || d.n_pages < 1) {
        snprintf(e->text, sizeof(e->text), "%d layers, %d kv heads, %d pages", d.n_layers, d.n_kv_heads, d.n_pages);
        return e->code;
    }
    const unsigned __int128 all = (unsigned __int128)pages_cell_bytes(d) * (unsigned)d.n_kv_heads * 2 * (unsigned)d.n_pages *
                                  (unsigned)d.n_layers;
    if (all > (uint64_t)INT64_MAX) {
        snprintf(e->text, sizeof(e->text), "the pages exceed 2^63 bytes");
        return e->code;
    }
    *bytes = (uint64_t)all;
    return e->code = FLLM_OK;
}

struct SeqPlan {
    int row0, n_new, len, pos0;  // first new row, new tokens, positions, first row of the positions
};

// The new tokens of a sequence in one page: n positions from `off` on, whose rows start at `row`.
struct PageTile {
    int off, n, row, page;
};

struct BatchPlan {
    int n_seqs = 0, n_rows = 0, n_pos = 0;
    int max_new = 0;                     // most new tokens of a sequence
    bool holes = false;                  // some page before the windows was given back
    std::vector<SeqPlan> seqs;
    std::vector<int32_t> first;          // where each sequence's pages start in `tables`; their number
    std::vector<int32_t> tables;         // the sequences' pages one after the other, 0 where there is none
    std::vector<PageTile> new_tiles;
    std::vector<uint8_t> uses;           // places that name a page (up to 2); zeros between calls
};

// Fills `p` from the arrays of fllm_batch_set, or says what is wrong with them.
inline int32_t batch_plan(const fllm_pages_desc& d, int window, int32_t n_seqs, const int32_t* n_new, const int32_t* lengths,
                          const int32_t* tables, int64_t ld, BatchPlan* p, BatchError* e) {
    p->n_seqs = p->n_rows = p->n_pos = p->max_new = 0;
    p->holes = false;
    p->seqs.clear();
    p->first.clear();
    p->new_tiles.clear();
    e->code = FLLM_E_ARG_RANGE;
    const int P = d.page_size;
    int64_t rows = 0, pos = 0, all = 0;
    int wide = 0;
    for (int i = 0; i < n_seqs; i++) {
        const int n = n_new[i], len = lengths[i];
        if (n < 0 || len < 0 || n > len || len > kPagesMaxLength) {
            snprintf(e->text, sizeof(e->text), "sequence %d: %d new tokens, length %d (at most %d)", i, n, len, kPagesMaxLength);
            return e->code;
        }
        const int blocks = (len + P - 1) / P;
        wide = blocks > wide ? blocks : wide;
        all += blocks;
        p->max_new = n > p->max_new ? n : p->max_new;
        rows += n;
        pos += len;
    }
    if (rows > INT32_MAX || pos > INT32_MAX) {
        e->code = FLLM_E_ARG;
        snprintf(e->text, sizeof(e->text), "%lld new rows, %lld positions: at most %d of each", (long long)rows, (long long)pos, INT32_MAX);
        return e->code;
    }
    if (ld < wide) {
        e->code = FLLM_E_ARG;
        snprintf(e->text, sizeof(e->text), "tables of %lld pages a sequence, %d are needed", (long long)ld, wide);
        return e->code;
    }
    p->uses.resize((size_t)d.n_pages);
    p->tables.assign((size_t)all, 0);  // at most n_pos
    struct Clear {  // what the tables name, not all pages: there may be millions
        BatchPlan* p;
        ~Clear() {
            for (const int32_t page : p->tables) p->uses[(size_t)page] = 0;
        }
    } clear{p};
    p->seqs.reserve((size_t)n_seqs);
    p->first.reserve((size_t)n_seqs + 1);
    int r = 0, q = 0, f = 0;
    for (int i = 0; i < n_seqs; i++) {
        const int n = n_new[i], len = lengths[i], blocks = (len + P - 1) / P;
        // the first position that any new token sees; without new tokens nothing is read
        const int64_t low = n ? (int64_t)(len - n) - window + 1 : len;
        const int first = low > 0 ? (int)(low / P) : 0;
        for (int k = 0; k < blocks; k++) {
            const int32_t page = tables[(int64_t)i * ld + k];
            if (page == -1 && k < first) {
                p->holes = true;
                continue;
            }
            if (page < 0 || page >= d.n_pages) {
                e->code = FLLM_E_ARG_RANGE;
                snprintf(e->text, sizeof(e->text), "sequence %d, block %d: page %d outside [0, %d)", i, k, page, d.n_pages);
                return e->code;
            }
            p->tables[(size_t)(f + k)] = page;
            if (p->uses[(size_t)page] < 2) p->uses[(size_t)page]++;
        }
        p->seqs.push_back({r, n, len, q});
        p->first.push_back(f);
        r += n;
        q += len;
        f += blocks;
    }
    p->first.push_back(f);
    for (int i = 0; i < n_seqs; i++) {
        const SeqPlan& s = p->seqs[(size_t)i];
        const int old = s.len - s.n_new;
        for (int k = old / P; s.n_new && k < (s.len + P - 1) / P; k++) {
            const int32_t page = p->tables[(size_t)(p->first[(size_t)i] + k)];
            if (p->uses[(size_t)page] > 1) {
                e->code = FLLM_E_ARG;
                snprintf(e->text, sizeof(e->text), "sequence %d writes page %d, which the tables name twice", i, page);
                return e->code;
            }
            const int lo = std::max(old, k * P), hi = std::min(s.len, k * P + P);
            p->new_tiles.push_back({lo - k * P, hi - lo, s.row0 + lo - old, page});
        }
    }
    p->n_seqs = n_seqs;
    p->n_rows = r;
    p->n_pos = q;
    return e->code = FLLM_OK;
}

// ---- the attention's work ------------------------------------------------------------------
// The rows of a sequence under one kv head are its new tokens times the head group: row r is token
// r / group, query head kvh * group + r % group. A tile is some of them; an item is a tile with a range
// [k0, k1) of the keys that its rows see, cut at multiples of kKeyStep. A tile of several items leaves a partial
// result of each, nsplit * nrows rows from `part` on per kv head, which the last item to finish joins.
struct AttnItem {
    int seq, row0, nrows, k0, k1, part, split, nsplit;
    int tok0, pos0, len, table;  // of the sequence: its first new row and that row's position, its length, its table's start
    int image;  // of a quantised cache's key step 0, counted in steps of kKeyStep (may be negative)
    int pad[3];
};
// Key steps of a sequence that are turned into images: n from position k0 on, the first being image `image`; positions
// outside [lo, len) count as nothing.
struct ImageItem {
    int table, len, lo, k0, n, image, pad[2];
};
constexpr int kKeyStep = 64;
// Classes of tiles: their rows, and the most items of one. The last class is that of sequences of many rows whose
// keys and values are turned into images first.
constexpr int kAttnClasses = 6, kAttnMany = 4, kAttnImage = 5;
constexpr int kAttnTile[kAttnClasses] = {4, 8, 16, 32, 128, 128};
constexpr int kAttnSplit[kAttnClasses] = {128, 128, 128, 128, 32, 32};
// Tiles from which images pay. One sequence of 4000, 8 kv heads, Q8_0, in us with images and without: heads of 128,
// BF16 rows: 2 tiles 57.0 and 49.0, 4 tiles 64.7 and 58.7, 8 tiles 76.7 and 73.1; heads of 256, F32 rows: 4 tiles 106.5 and
// 90.5, 8 tiles 200 and 216. Two of 2000, Q4_0, F32 rows: 8 tiles 103.6 and 103.2.
constexpr int kImageTiles = 8;
constexpr int kImageRun = 4;    // key steps of an image item
constexpr uint64_t kImageBytes = (uint64_t)4 << 30;  // a batch's images at most; beyond, every tile turns the codes itself
// bytes of the images of one kv head's key step; wide: F32 rows of q or out
inline uint64_t attend_image_bytes(int hd, bool wide) {
    return (uint64_t)(hd <= 64 ? 64 : hd <= 128 ? 128 : 256) * kKeyStep * 2 * 2 * (wide ? 2 : 1);
}

struct AttnPlan {
    std::vector<AttnItem> items[kAttnClasses];  // tiles of up to kAttnTile[c] rows
    int64_t part_rows = 0;           // partial rows per kv head
    std::vector<ImageItem> image_items;
    int64_t images = 0;              // key steps that they make, per kv head
};

// Items of the tiles of class c of sequence i, each of at most `steps` steps of keys where the splits allow it.
inline void attn_items(const SeqPlan& s, int i, int table, int image, int group, int window, int c, int64_t steps,
                       std::vector<AttnItem>* out, int64_t* part_rows) {
    const int64_t rows = (int64_t)s.n_new * group;
    const int tile = kAttnTile[c];
    for (int64_t r = 0; r < rows; r += tile) {
        const int n = (int)std::min<int64_t>(tile, rows - r);
        const int pos0 = s.len - s.n_new;
        const int64_t low = (int64_t)pos0 + r / group - window + 1;
        const int g0 = low > 0 ? (int)(low / kKeyStep) : 0;
        const int last = pos0 + (int)((r + n - 1) / group);
        const int g1 = last / kKeyStep + 1;
        const int nsplit = (int)std::min<int64_t>(kAttnSplit[c], (g1 - g0 + steps - 1) / steps), per = (g1 - g0 + nsplit - 1) / nsplit;
        const int used = (g1 - g0 + per - 1) / per;
        for (int k = 0; k < used; k++)
            out->push_back({i, (int)r, n, (g0 + k * per) * kKeyStep, std::min((g0 + (k + 1) * per) * kKeyStep, last + 1),
                            (int)*part_rows, k, used, s.row0, pos0, s.len, table, image, {0, 0, 0}});
        if (used > 1) *part_rows += (int64_t)used * n;
    }
}

struct AttnCount {
    int64_t items = 0, steps = 0, longest = 0;
};
// What a sequence's tiles of class c become under one kv head with at most `steps` steps of keys an item.
inline void attn_count(const SeqPlan& s, int group, int window, int c, int64_t steps, AttnCount* n) {
    const int64_t rows = (int64_t)s.n_new * group;
    for (int64_t r = 0; r < rows; r += kAttnTile[c]) {
        const int64_t low = (int64_t)s.len - s.n_new + r / group - window + 1;
        const int64_t last = (int64_t)s.len - s.n_new + (std::min<int64_t>(rows, r + kAttnTile[c]) - 1) / group;
        const int64_t all = last / kKeyStep + 1 - (low > 0 ? low / kKeyStep : 0);
        const int64_t k = std::min<int64_t>(kAttnSplit[c], (all + steps - 1) / steps);
        n->items += k;
        n->steps += all;
        n->longest = std::max(n->longest, (all + k - 1) / k);
    }
}

// Key steps an item of few rows should have at least: one that is cut into n parts ends when its workgroup has read
// S / n steps and the one that joins them n partial results, both as fast as one CU can; S steps of rows r and e bytes an
// element balance at sqrt(S r / (16 e)). One sequence, 4 rows, Q8_0, in us with 2, 4 and 8 steps an item: 518 positions
// 8.8, 9.4, 11.3; 2048: 9.5, 9.7, 11.8; 4096: 12.3, 10.5, 12.0; 8192: 14.2, 14.2, 13.1. 4 sequences of 2000, 20
// rows, F16: 20.8, 19.2, 20.3; 7 rows, Q8_0: 10.5, 11.4, 14.4, so that fewer than 4 are left alone. Longer sequences
// fill all CUs with 8 steps and more.
inline int64_t join_steps(const SeqPlan& s, int group, int window, int c, bool quant) {
    AttnCount n;
    attn_count(s, group, window, c, 1, &n);
    const int64_t rows = std::min<int64_t>((int64_t)s.n_new * group, kAttnTile[c]), tiles = ((int64_t)s.n_new * group + kAttnTile[c] - 1) / kAttnTile[c];
    const double best = std::sqrt((double)(n.steps / tiles * rows) / (quant ? 16.0 : 32.0));
    return best < 4.0 ? 0 : std::min<int64_t>(8, 2 * (int64_t)(best / 2 + 0.5));
}

// The items of a batch on a device of n_cu CUs. False where they or their partial rows are too many.
inline bool attn_plan(const BatchPlan& b, int n_heads, int n_kv, int head_dim, bool quant, int window, int n_cu, AttnPlan* p) {
    const int group = n_heads / n_kv;
    p->part_rows = p->images = 0;
    p->image_items.clear();
    const auto imaged = [&](const SeqPlan& s) { return quant && (int64_t)s.n_new * group > (kImageTiles - 1) * kAttnTile[kAttnMany]; };
    const auto first_image = [&](const SeqPlan& s) { return std::max<int64_t>(0, (int64_t)s.len - s.n_new - window + 1) / kKeyStep; };
    uint64_t steps_imaged = 0;
    for (const SeqPlan& s : b.seqs)
        if (imaged(s)) steps_imaged += (uint64_t)((s.len - 1) / kKeyStep + 1 - first_image(s));
    const bool images = steps_imaged * (uint64_t)n_kv * attend_image_bytes(head_dim, true) <= kImageBytes;
    // the smallest tile that holds the sequence's rows; an F16 cache has no use for the two smallest (pages_attend.hpp)
    const auto class_of = [&](const SeqPlan& s) {
        const int64_t rows = (int64_t)s.n_new * group;
        int c = quant ? 0 : 2;
        while (c < kAttnMany && rows > kAttnTile[c]) c++;
        // 17 to 32 rows: two tiles of 16, except where one pass over the keys is faster (8 sequences of 4000, 20 and 32
        // rows, in us in one pass and in two: F16 38.3 and 41.5, 41.2 and 41.5; Q8_0 30.9 and 31.4, 33.8 and 31.9).
        // Wide heads leave no registers for it.
        if (c == 3 && (quant || head_dim > 128)) c = 2;
        return images && imaged(s) ? kAttnImage : c;
    };
    // two workgroups are resident on a CU, one of heads wider than 128
    const int64_t slots = (head_dim > 128 ? 1 : 2) * (int64_t)n_cu;
    // Few rows: the shortest items whose workgroups all start at once (two key steps at
    // least), so that the longest one is as short as it can be.
    int64_t few = 2, hi = kPagesMaxLength / kKeyStep + 1;
    while (few < hi) {
        const int64_t mid = (few + hi) / 2;
        AttnCount n;
        for (const SeqPlan& s : b.seqs)
            if (class_of(s) < kAttnMany) attn_count(s, group, window, class_of(s), mid, &n);
        if (n.items * n_kv <= slots) hi = mid;
        else few = mid + 1;
    }
    // Many rows: tiles whole, or cut where that ends sooner. Longest first, a grid of more items than slots ends
    // about half a longest item after the mean; a part of a tile costs about 3 steps more (its partial rows).
    const auto ends = [&](int64_t steps, AttnCount* n) {
        for (const SeqPlan& s : b.seqs)
            if (class_of(s) >= kAttnMany) attn_count(s, group, window, kAttnMany, steps, n);
        return n->items * n_kv <= slots ? (double)n->longest
                                        : (double)(n->steps + 3 * n->items) * n_kv / (double)slots + 0.5 * (double)n->longest;
    };
    AttnCount whole;
    int64_t many = hi = kPagesMaxLength / kKeyStep + 1;
    double best = ends(many, &whole);
    for (int k = 1; k <= 3 && whole.items; k++) {
        const int64_t steps = std::max<int64_t>(4, whole.steps * n_kv / (slots * k) + 1);
        AttnCount n;
        const double t = ends(steps, &n) + 3.0;
        if (t < 0.95 * best) best = t, many = steps;
    }
    for (auto& v : p->items) v.clear();
    for (int i = 0; i < b.n_seqs; i++) {
        const SeqPlan& s = b.seqs[(size_t)i];
        const int c = class_of(s);
        int64_t image = 0;
        if (s.n_new && c == kAttnImage) {
            const int64_t low = std::max<int64_t>(0, (int64_t)s.len - s.n_new - window + 1);
            const int g0 = (int)first_image(s), g1 = (s.len - 1) / kKeyStep + 1;
            image = p->images - g0;
            for (int g = g0; g < g1; g += kImageRun)
                p->image_items.push_back({b.first[(size_t)i], s.len, (int)low, g * kKeyStep, std::min(kImageRun, g1 - g), (int)(image + g), {0, 0}});
            p->images += g1 - g0;
        }
        if (s.n_new)
            attn_items(s, i, b.first[(size_t)i], (int)image, group, window, c, c >= kAttnMany ? many : std::max(few, join_steps(s, group, window, c, quant)),
                       &p->items[c], &p->part_rows);
        if (p->part_rows > INT32_MAX / n_kv) return false;
    }
    if ((int64_t)p->image_items.size() * n_kv >= 1 << 23) return false;
    for (auto& v : p->items) {
        if ((int64_t)v.size() * n_kv >= 1 << 23) return false;  // a grid ends at 2^32 threads
        // the long ones first: the short ones fill the end
        std::stable_sort(v.begin(), v.end(), [](const AttnItem& x, const AttnItem& y) { return x.k1 - x.k0 > y.k1 - y.k0; });
    }
    return true;
}

}  // namespace fllm
