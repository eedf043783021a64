// pages_attend.hpp — the kernels that attend from new tokens to the pages of their sequences; one translation
// unit per cache type (pages_attend_f16.hip, pages_attend_q8_0.hip, pages_attend_q4_0.hip) instantiates them.
//
// Mathematics. o = sum_j w_j v_j / sum_j w_j, w_j = exp(s_j - m), in one pass over the keys with the
// running maximum m: whatever has been summed is multiplied by exp(m_old - m_new) when m grows. The
// products run on the fp16 matrix cores, transposed: S^T = K Q^T and O^T = V^T P^T, so that a lane
// holds one query's scores (column l & 15 of the tile) and the weights are, as they lie in the score
// registers, the second product's operand. All sums are f32.
//
// Factors. Every row of q is scaled by a power of two (largest magnitude into [2^14, 2^15)) and rounded
// to fp16, for F32 rows as a high and a low half that together keep 22 bits (NP = 2: two products in place of
// one). K and V enter exactly: the halves of an F16 cache, the codes of a quantised one as
// integers, whose scales are applied in f32: to the scores block by block, and to the weights before they are
// rounded (as one or two halves), so that a V block's product is weights-times-scales by codes.
//
// k_attend_few: up to 16 TM rows (decoding, drafted tokens), bound by the bytes of K and V. A wave
// takes steps of 64 keys (32 of an F16 cache) for all rows straight from the pages into registers: the page
// layouts (fllm.h) are such that 8 consecutive elements of an operand are contiguous in memory, so
// there is no LDS stage and no barrier in the loop. The four waves of a workgroup take turns at the
// steps of an item; their results meet in LDS, and those of a tile's items in memory, joined by
// the item that finishes last (write-through stores and a counter, as the decode attention of
// attn_body.hpp, so no second launch). Measured: 64 sequences of 200 to 8000 positions, 28 over 4 heads of 128,
// Q8_0: 183 MB in 47 us (3.9 TB/s); one of 131071, 32 over 8 heads, Q4_0: 151 MB in 55 us, of 262141: 302 MB in 95 us;
// Q8_0 of that length 5.4 TB/s, F16 5.8 (a large read reaches 5.6): what is over that rate's time is, at any length,
// 10 to 14 us of launch, first loads and join, and for Q4_0 the turning of codes into halves.
#pragma once

#include <type_traits>

#include "attn_body.hpp"
#include "pages.hpp"
#include "pages_plan.hpp"

namespace fllm {

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
enum { DPP_ROR4 = 0x124, DPP_ROR8 = 0x128 };  // rotation within 16 lanes
constexpr float kNoScore = -3e38f;  // the running maximum before any key: below finite scores of any size that q k may have

union H8 {
    h8 v;
    h2 p[4];
    uint32_t u[4];
};

// The scale of the scores in two parts: its sign, which goes into q, and its magnitude, never zero (a masked score is
// -inf, times zero it would be a NaN): a scale of zero makes q zero.
__device__ __forceinline__ float scale_sign(float s) { return s < 0.0f ? -1.0f : s > 0.0f ? 1.0f : 0.0f; }
__device__ __forceinline__ float scale_size(float s, int e, float softcap) {
    return fminf(fmaxf(ldexpf(s == 0.0f ? 1.0f : fabsf(s), -e) * (softcap > 0.0f ? 1.0f / softcap : kLog2e), 1e-37f), 3e38f);
}

// 4 bytes, each code + 128 or nibble, as fp16 integers: 0x6400 | byte is 1024 + byte exactly
template <int OFF>
__device__ __forceinline__ void bytes_to_half(uint32_t w, uint32_t* out) {
    const h2 off = {(_Float16)OFF, (_Float16)OFF};
    union { uint32_t u; h2 h; } a, b;
    a.u = __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u);
    b.u = __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u);
    a.h = a.h - off;
    b.h = b.h - off;
    out[0] = a.u;
    out[1] = b.u;
}

// A lane's 8 operand elements out of what it loads of a cell: 16, 8 or 4 bytes.
template <int TYPE> struct Frag;
template <> struct Frag<FLLM_TYPE_F16> {
    u4 w;
    __device__ __forceinline__ void load(const uint8_t* p) { w = *(const u4*)p; }
    __device__ __forceinline__ h8 half() const {
        H8 r;
        for (int i = 0; i < 4; i++) r.u[i] = w[i];
        return r.v;
    }
};
template <> struct Frag<FLLM_TYPE_Q8_0> {
    u2 w;
    __device__ __forceinline__ void load(const uint8_t* p) { w = *(const u2*)p; }
    __device__ __forceinline__ h8 half() const {
        H8 r;
        bytes_to_half<1152>(w.x ^ 0x80808080u, r.u);
        bytes_to_half<1152>(w.y ^ 0x80808080u, r.u + 2);
        return r.v;
    }
};
template <> struct Frag<FLLM_TYPE_Q4_0> {  // elements 4 g .. + 3 in the low halves, 16 + 4 g .. in the high ones
    uint32_t w;
    __device__ __forceinline__ void load(const uint8_t* p) { w = *(const uint32_t*)p; }
    __device__ __forceinline__ h8 half() const {
        H8 r;
        bytes_to_half<1032>(w & 0x0F0F0F0Fu, r.u);
        bytes_to_half<1032>(w >> 4 & 0x0F0F0F0Fu, r.u + 2);
        return r.v;
    }
};

__device__ __forceinline__ uint32_t bits(h2 h) {
    union { uint32_t u; h2 h; } c;
    c.h = h;
    return c.u;
}

// e such that 2^e brings a largest magnitude `top` into [2^14, 2^15); 0 for zeros and what is no number
__device__ __forceinline__ int row_exponent(float top) {
    if (!(top > 0.0f && top < INFINITY)) return 0;
    const int e = 15 - __builtin_amdgcn_frexp_expf(top);  // top = f 2^k, f in [1/2, 1): e = 15 - k
    return e > 120 ? 120 : e;
}

// 8 codes (two words) as fp16 integers; Q4_0: of the low (half 0) or high nibbles
template <int TYPE>
__device__ __forceinline__ H8 codes8(uint32_t a, uint32_t b, int half) {
    H8 r;
    if (TYPE == FLLM_TYPE_Q8_0) {
        bytes_to_half<1152>(a ^ 0x80808080u, r.u);
        bytes_to_half<1152>(b ^ 0x80808080u, r.u + 2);
    } else {
        bytes_to_half<1032>(a >> 4 * half & 0x0F0F0F0Fu, r.u);
        bytes_to_half<1032>(b >> 4 * half & 0x0F0F0F0Fu, r.u + 2);
    }
    return r;
}

// Mixed-precision multiply-adds on half SEL of a word: a b of two halves, a b of a half and a float, x - a.
template <int SEL>
__device__ __forceinline__ float mix_mul(uint32_t a, uint32_t b) {
    float r;
    if (SEL) asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel:[1,1,0] op_sel_hi:[1,1,0]" : "=v"(r) : "v"(a), "v"(b));
    else asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel_hi:[1,1,0]" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
template <int SEL>
__device__ __forceinline__ float mix_scale(uint32_t a, float b) {
    float r;
    if (SEL) asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(a), "v"(b));
    else asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
template <int SEL>
__device__ __forceinline__ float mix_rest(uint32_t a, float x) {
    float r;
    if (SEL) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(a), "v"(x));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(a), "v"(x));
    return r;
}

// x and y as a high and a low half each
__device__ __forceinline__ void split2(float x, float y, h2* hi, h2* lo) {
    union { __fp16 __attribute__((ext_vector_type(2))) c; h2 h; uint32_t u; } a, b;
    a.c = __builtin_amdgcn_cvt_pkrtz(x, y);
    b.c = __builtin_amdgcn_cvt_pkrtz(mix_rest<0>(a.u, x), mix_rest<1>(a.u, y));
    *hi = a.h;
    *lo = b.h;
}

// x as fp16 halves: one rounded to nearest, or a high and a low one (both cut, together 21 to 22 bits)
template <int NP>
__device__ __forceinline__ void split4(const f4 x, h2 out[NP][2]) {
    for (int i = 0; i < 2; i++) {
        if (NP == 1) out[0][i] = h2{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
        else split2(x[2 * i], x[2 * i + 1], &out[0][i], &out[NP - 1][i]);
    }
}
// x + the sum of 8 halves: what the product with V weighs with, where the weights are rounded to one half
__device__ __forceinline__ float add_halves(h8 w, float x) {
    H8 h;
    h.v = w;
    const h2 one = {(_Float16)1.0f, (_Float16)1.0f};
    for (int i = 0; i < 4; i++) x = __builtin_amdgcn_fdot2(h.p[i], one, x, false);
    return x;
}

template <int NP>
__device__ __forceinline__ void split8(const float x[8], h8 out[NP]) {
    h2 a[NP][2], b[NP][2];
    split4<NP>(f4{x[0], x[1], x[2], x[3]}, a);
    split4<NP>(f4{x[4], x[5], x[6], x[7]}, b);
    for (int n = 0; n < NP; n++) {
        H8 h;
        h.p[0] = a[n][0], h.p[1] = a[n][1], h.p[2] = b[n][0], h.p[3] = b[n][1];
        out[n] = h.v;
    }
}

// cap tanh(us s) of a lane's N scores. Near zero the quotient (1 - t) / (1 + t), t = exp(-2 |x|), cancels: below 1/10
// a series to x^5 is exact to 6e-8, and where a wave's scores are all that small it is all that runs (SERIES).
template <int N, bool SERIES, typename V>
__device__ __forceinline__ void softcap_n(V& s, float us, float cap) {
    float top = 0.0f;
    for (int i = 0; i < N; i++) {
        s[i] *= us;
        top = fmaxf(top, fabsf(s[i]));
    }
    if (SERIES && !__any(top >= 0.1f)) {
        for (int i = 0; i < N; i++) {
            const float y = s[i] * s[i];
            s[i] *= cap * fmaf(y, fmaf(y, 2.0f / 15.0f, -1.0f / 3.0f), 1.0f);
        }
        return;
    }
    for (int i = 0; i < N; i++) {
        const float x = s[i], y = x * x;
        const float p = x * fmaf(y, fmaf(y, 2.0f / 15.0f, -1.0f / 3.0f), 1.0f);
        const float t = __builtin_amdgcn_exp2f(-2.0f * kLog2e * fabsf(x));
        const float q = copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), x);
        const uint32_t big = fabsf(x) < 0.1f ? 0u : 0xFFFFFFFFu;  // selected by bits: no branch per score
        s[i] = cap * __uint_as_float((__float_as_uint(q) & big) | (__float_as_uint(p) & ~big));
    }
}
// Weights are exp2(us s - m) in one rounding. Where a maximum m is so large that its own rounding shows (2^-24 of
// 2^20 and more), the products are rounded first, so that the largest score's weight is 1; m is that rounded product.
__device__ __forceinline__ bool is_far(float m) { return __any(m > kNoScore && fabsf(m) >= 0x1p20f); }

__device__ __forceinline__ f4 load_row4(const RowsView& r, int64_t i) {
    if (r.type == FLLM_TYPE_F32) return *(const f4*)(r.p + 4 * i);
    const u2 u = *(const u2*)(r.p + 2 * i);
    f4 v;
    if (r.type == FLLM_TYPE_F16) {
        union { uint32_t u; h2 h; } a, b;
        a.u = u.x;
        b.u = u.y;
        v = f4{(float)a.h.x, (float)a.h.y, (float)b.h.x, (float)b.h.y};
    } else {
        v = f4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u)};
    }
    return v;
}
__device__ __forceinline__ void store_row4(const RowsView& r, int64_t i, f4 v) {
    if (r.type == FLLM_TYPE_F32) {
        *(f4*)(r.p + 4 * i) = v;
        return;
    }
    uint32_t h[4];
    for (int e = 0; e < 4; e++) {
        union { _Float16 h; uint16_t u; } c;
        c.h = (_Float16)v[e];
        h[e] = r.type == FLLM_TYPE_F16 ? c.u : bf16_round(v[e]);
    }
    *(u2*)(r.p + 2 * i) = u2{h[0] | h[1] << 16, h[2] | h[3] << 16};
}

struct AttnArgsP {
    PagesView pg;
    const int* tables;
    const AttnItem* items;
    int group, window;
    RowsView q, out;
    float scale, softcap;
    float *part_o, *part_ml;
    unsigned* cnt;
    void* images;         // SRC_IMAGE
    float* image_units;
};

// Counts this workgroup's partial rows, whose stores were all issued before, as there; true for the workgroup that
// completes the tile's `n`, which also leaves the counter at zero for the next call.
__device__ __forceinline__ bool last_of_tile(unsigned* cnt, int n, int* s_last) {
    wt_complete();
    __syncthreads();
    if (threadIdx.x == 0)
        *s_last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(n - 1);
    __syncthreads();
    if (*s_last && threadIdx.x == 0) st_wt_u(cnt, 0u);
    return *s_last != 0;
}

// Joins a tile's partial rows [split][row] (ro: head_dim floats, rml: max and sum) into out. w: MAXS floats a row.
template <int MAXS, int NT = 256>
__device__ __forceinline__ void join_parts(const AttnArgsP& a, const AttnItem& it, int kvh, __amdgpu_buffer_rsrc_t ro,
                                           __amdgpu_buffer_rsrc_t rml, float* w) {
    constexpr int N = (MAXS + 63) / 64;
    const int lane = threadIdx.x & 63, hd = a.pg.hd;
    // weights of the parts, a wave per row: exp2(m - max) / sum
    for (int row = threadIdx.x >> 6; row < it.nrows; row += NT / 64) {
        float m1[N], l1[N], top = kNoScore, l = 0.0f;
        for (int i = 0; i < N; i++) {
            const int k = lane + 64 * i;
            const float2 v = ld_wt2(rml, (uint32_t)((k < it.nsplit ? k : 0) * it.nrows + row) * 8);
            m1[i] = k < it.nsplit ? v.x : kNoScore;
            l1[i] = k < it.nsplit ? v.y : 0.0f;
            top = fmaxf(top, m1[i]);
        }
        top = wave_max(top);
        for (int i = 0; i < N; i++) {
            m1[i] = __builtin_amdgcn_exp2f(m1[i] - top);
            l += m1[i] * l1[i];
        }
        const float inv = 1.0f / wave_sum(l);
        for (int i = 0; i < N; i++)  // zeros past the end
            if (lane + 64 * i < MAXS) w[row * MAXS + lane + 64 * i] = lane + 64 * i < it.nsplit ? m1[i] * inv : 0.0f;
    }
    __syncthreads();
    for (int u = threadIdx.x; u < it.nrows * (hd / 4); u += NT) {
        const int row = u / (hd / 4), d = u % (hd / 4) * 4;
        f4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < it.nsplit; k0 += 16) {  // 16 loads on their way; those past the end read zeros
            float4 v[16];
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = ld_wt4(ro, (uint32_t)(((k0 + i) * it.nrows + row) * hd + d) * 4);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float f = w[row * MAXS + k0 + i];
                acc += f * f4{v[i].x, v[i].y, v[i].z, v[i].w};
            }
        }
        const int tr = it.row0 + row, tok = tr / a.group, head = kvh * a.group + tr % a.group;
        store_row4(a.out, (int64_t)(it.tok0 + tok) * a.out.ld + (int64_t)head * hd + d, acc);
    }
}

// Wide heads take the registers of two waves: one wave a SIMD then has as many bytes on their way.
//
// RC is the tile's rows: 4, 8 or 16 (with a second tile TM = 2). One and 32 sequences of 4000, 32 over 8 heads, Q8_0, in us
// with 4 columns a row group, 8 and 16: 9.1, 9.6, 9.2 and 56.2, 59.9, 60.4; 28 over 4 heads with 8 and 16: 10.0, 9.8 and
// 35.6, 37.1.
//
// Columns. A quantised cache has a scale per key and block of 32 elements, so that every block needs operands of its
// own. Tiles of RC < 16 rows leave columns of the matrix tiles over: the rows are repeated in SUB groups of columns and
// group j works on the blocks [j BPS, (j + 1) BPS) alone. Its q is zero in the other blocks, so one chain of products
// gives each column its block's dot product, to be scaled once and summed over the groups; its weights are
// multiplied by its own blocks' scales, and of each product with V only the columns whose group the block belongs
// to are kept. A lane then loads and applies BPS scales a key in place of NB.
template <int TYPE, int HDP, int NP, int TM, int RC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HDP > 128 ? 1 : 2, HDP > 128 ? 1 : 2))) void k_attend_few(AttnArgsP a) {
    constexpr int NB = HDP / 32, ND = HDP / 16;      // blocks of 32 elements, tiles of 16
    constexpr bool QUANT = TYPE != FLLM_TYPE_F16;
    // runs of 32 keys a step: 16 bytes of V a lane, 8 where registers are short
    constexpr int JN = QUANT && HDP <= 128 && RC < 16 ? 2 : 1;
    constexpr int STEP = 32 * JN, RUN = 8 * JN;      // keys a step, consecutive keys a lane holds
    constexpr int SUB = !QUANT || 16 / RC < 1 ? 1 : 16 / RC < NB ? 16 / RC : NB, BPS = NB / SUB;
    constexpr int NV = TYPE == FLLM_TYPE_Q4_0 ? NB : ND;  // loads of V a step (one byte row holds two elements in Q4_0)
    constexpr bool QLDS = HDP * TM >= 256;           // q stays in LDS where registers are short
    __shared__ union {
        _Float16 q[NP][16 * TM][HDP + 8];  // the rows' halves
        float o[4][16][HDP + 4];           // a row tile's result of each wave
        float w[kAttnSplit[0] * 32];       // weights of the parts
    } sm;
    __shared__ float s_m[4][16], s_l[4][16], s_scale[16 * TM];
    __shared__ int s_last;

    const int kvh = blockIdx.x % a.pg.nkv;
    const AttnItem it = a.items[blockIdx.x / a.pg.nkv];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int hd = a.pg.hd, nb = hd >> 5, lp = a.pg.page_log2, P = 1 << lp;
    const int pos0 = it.pos0;
    const int* table = a.tables + it.table;
    const int last_block = (it.len - 1) >> lp;

    // this lane's row of a tile, and the group of columns that it is in
    const int cq = RC < 16 ? col % RC : col, sub = RC < 16 ? col / RC % SUB : 0;
    constexpr int ksub = RUN;  // keys of a lane group
    // K: row col of tile (j, t) is key ksub (col >> 2) + 8 j + 4 t + (col & 3) of the step; V: this lane holds the keys
    // ksub g .. + RUN. Both lie in one page each; past the table's end the last page stands in. A step's K is loaded
    // as soon as the step before has its scores, its V once the step before is added up, so that both are on their way
    // through the other half of a step; the page numbers are a step ahead of them.
    constexpr int KB = TYPE == FLLM_TYPE_F16 ? 64 : TYPE == FLLM_TYPE_Q8_0 ? 32 : 16;  // bytes of a block's codes
    constexpr int VW = TYPE == FLLM_TYPE_F16 ? 4 : 2 * JN, VE = TYPE == FLLM_TYPE_F16 ? 2 : 1;
    typedef uint32_t uv __attribute__((ext_vector_type(VW)));
    Frag<TYPE> kf[2 * JN][NB];
    u4 ks[QUANT ? BPS : 1][JN], vs[QUANT ? BPS : 1][JN];  // scales of this lane's keys, 8 to a vector
    uv vf[NV];                                            // 8 halves, or the codes of this lane's keys
    int tk, tv;                                           // pages of the next step
    uint64_t cv;                                          // the step's cell for this lane's keys
    const auto pages_at = [&](int k0) {
        tk = table[min((k0 + ksub * (col >> 2)) >> lp, last_block)];
        tv = table[min((k0 + ksub * g) >> lp, last_block)];
    };
    const auto load_k = [&](int k0) {
        const int kk = k0 + ksub * (col >> 2), pv = (k0 + ksub * g) & (P - 1);
        const uint64_t ck = ((uint64_t)(uint32_t)tk * a.pg.nkv + kvh) * a.pg.cell;
        cv = ((uint64_t)(uint32_t)tv * a.pg.nkv + kvh) * a.pg.cell;
        const uint8_t* kp = a.pg.k + ck + (uint32_t)(((kk & (P - 1)) + (col & 3)) * KB + g * (KB / 4));
#pragma unroll
        for (int t = 0; t < 2 * JN; t++)
#pragma unroll
            for (int c = 0; c < NB; c++) kf[t][c].load(kp + (uint32_t)(((c < nb ? c : 0) * P + 4 * t) * KB));
        if (QUANT)
#pragma unroll
            for (int c = 0; c < BPS; c++)
                for (int i = 0; i < JN; i++) {
                    const int blk = sub * BPS + c;
                    ks[c][i] = *(const u4*)(a.pg.k + cv + a.pg.scale_off + (uint32_t)(2 * ((blk < nb ? blk : 0) * P + pv)) + 16 * i);
                }
    };
    const auto load_v = [&](int k0) {
        const int pv = (k0 + ksub * g) & (P - 1);
        if (QUANT)
#pragma unroll
            for (int c = 0; c < BPS; c++)
                for (int i = 0; i < JN; i++) {
                    const int blk = sub * BPS + c;
                    vs[c][i] = *(const u4*)(a.pg.v + cv + a.pg.scale_off + (uint32_t)(2 * ((blk < nb ? blk : 0) * P + pv)) + 16 * i);
                }
        const uint8_t* vp = a.pg.v + cv + (uint32_t)((col * P + pv) * VE);
#pragma unroll
        for (int d = 0; d < NV; d++)
            vf[d] = *(const uv*)(vp + (uint32_t)((d < (TYPE == FLLM_TYPE_Q4_0 ? nb : 2 * nb) ? d : 0) * 16 * P * VE));
    };
    const int first = it.k0 + wave * STEP;
    if (first < it.k1) {
        pages_at(first);
        load_k(first);
        load_v(first);
        pages_at(first + 4 * STEP < it.k1 ? first + 4 * STEP : first);
    }

    // q as fp16 halves in LDS, 16 lanes a row: every row scaled by the power of two 2^e that brings its largest
    // magnitude into [2^14, 2^15); zeros for the rows and elements that are not there
#pragma unroll
    for (int m = 0; m < TM; m++) {
        const int r = 16 * m + (threadIdx.x >> 4), l16 = threadIdx.x & 15;
        const bool live = r < it.nrows;
        const int row = it.row0 + (live ? r : 0), tok = row / a.group, head = kvh * a.group + row % a.group;
        const int64_t at = (int64_t)(it.tok0 + tok) * a.q.ld + (int64_t)head * hd;
        f4 x[HDP / 64];
#pragma unroll
        for (int i = 0; i < HDP / 64; i++) {
            const int d = 4 * l16 + 64 * i;
            x[i] = load_row4(a.q, at + (d < hd ? d : 0));
            if (!live || d >= hd) x[i] = f4{0.f, 0.f, 0.f, 0.f};
        }
        float top = 0.0f;
        for (int i = 0; i < HDP / 64; i++)
            for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(x[i][e]));
        for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
        const int e = row_exponent(top);
#pragma unroll
        for (int i = 0; i < HDP / 64; i++) {
            const f4 y = x[i] * ldexpf(scale_sign(a.scale), e);
            h2 h[NP][2];
            split4<NP>(y, h);
            for (int n = 0; n < NP; n++) *(u2*)&sm.q[n][r][4 * l16 + 64 * i] = u2{bits(h[n][0]), bits(h[n][1])};
        }
        if (l16 == 0) s_scale[r] = scale_size(a.scale, e, a.softcap);
    }
    __syncthreads();
    // this lane's query of each row tile: its position (-1 where there is no row), what undoes its scaling
    int pos[TM], low[TM];  // and the first position that it sees
    float unscale[TM];
    h8 qr[QLDS ? 1 : TM][QLDS ? 1 : NB][NP];
    const auto q_frag = [&](int m, int c, int n) {
        const _Float16* p = &sm.q[n][16 * m + cq][32 * c];
        H8 f;  // the elements that Frag's 8 stand for
        if (TYPE != FLLM_TYPE_Q4_0) {
            f.v = *(const h8*)(p + 8 * g);
        } else {
            *(u2*)&f.u[0] = *(const u2*)(p + 4 * g);
            *(u2*)&f.u[2] = *(const u2*)(p + 16 + 4 * g);
        }
        if (SUB > 1 && c / BPS != sub) f.u[0] = f.u[1] = f.u[2] = f.u[3] = 0;
        return f.v;
    };
#pragma unroll
    for (int m = 0; m < TM; m++) {
        const int r = 16 * m + cq;
        pos[m] = r < it.nrows ? pos0 + (it.row0 + r) / a.group : -1;
        low[m] = (int)max((int64_t)pos[m] - a.window + 1, (int64_t)INT_MIN);
        unscale[m] = s_scale[r];
        if (!QLDS) {
#pragma unroll
            for (int c = 0; c < NB; c++)
                for (int n = 0; n < NP; n++) qr[m][c][n] = q_frag(m, c, n);
        }
    }
    const auto q_of = [&](int m, int c, int n) { return QLDS ? q_frag(m, c, n) : qr[QLDS ? 0 : m][QLDS ? 0 : c][n]; };
    f4 o[TM][ND];
    float mx[TM], sum[TM];
    int vexp = -30;  // quantised: o is in units of 2^(vexp - 14), vexp at least the exponent of any scale so far (2^-24 and up, or zeros)
    for (int m = 0; m < TM; m++) {
        mx[m] = kNoScore;
        sum[m] = 0.0f;
        for (int d = 0; d < ND; d++) o[m][d] = f4{0.f, 0.f, 0.f, 0.f};
    }
    // Elements past head_dim stand for those of block 0 in K (times zeros of q) and V (results dropped).
    // keys that every row sees need no mask: [all_lo, all_hi)
    const int last_pos = pos0 + (it.row0 + it.nrows - 1) / a.group;
    const int64_t all_lo = (int64_t)last_pos - a.window + 1, all_hi = pos0 + it.row0 / a.group + 1;
    const int64_t any_lo = all_hi - a.window;  // the first key that any row sees

    for (int k0 = first; k0 < it.k1; k0 += 4 * STEP) {
        if (QLDS) asm volatile("" ::: "memory");  // or its reads would be kept in registers across the loop
        const int kv = k0 + ksub * g;
        // unconditionally, or the waits for this step's loads would wait for the next one's too: the last step again
        const int next = k0 + 4 * STEP < it.k1 ? k0 + 4 * STEP : k0;
        float s[TM][RUN];
#pragma unroll
        for (int m = 0; m < TM; m++)
#pragma unroll
            for (int t = 0; t < 2 * JN; t++) {
                f4 acc = {0.f, 0.f, 0.f, 0.f};
                if (QUANT) {
#pragma unroll
                    for (int p = 0; p < BPS; p++) {
                        f4 b = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = 0; j < SUB; j++) {
                            const h8 kh = kf[t][j * BPS + p].half();
                            for (int n = NP - 1; n >= 0; n--) b = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, q_of(m, j * BPS + p, n), b, 0, 0, 0);
                        }
                        for (int e = 0; e < 4; e++) {
                            union { uint32_t u; h2 h; } d;
                            d.u = ks[p][t >> 1][2 * (t & 1) + (e >> 1)];
                            acc[e] = fmaf(b[e], (float)(e & 1 ? d.h.y : d.h.x), acc[e]);
                        }
                    }
                    for (int e = 0; e < 4; e++) {  // over the groups of columns
                        if (SUB > 1 && SUB * RC > 8) acc[e] += dpp<DPP_ROR8>(0.0f, acc[e]);
                        if (SUB > 1 && RC == 4) acc[e] += dpp<DPP_ROR4>(0.0f, acc[e]);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < NB; c++)
                        for (int n = NP - 1; n >= 0; n--)
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][c].half(), q_of(m, c, n), acc, 0, 0, 0);
                }
                for (int e = 0; e < 4; e++) s[m][4 * t + e] = acc[e];
            }
        load_k(next);

        const bool edge = k0 < all_lo || k0 + STEP > all_hi;
        if (edge) {
            // what lies outside the sequence may be anything: no scale and no half of it may be a NaN
            for (int i = 0; i < RUN; i++) {
                const bool in = kv + i >= any_lo && kv + i < it.len;
                if (QUANT) {
                    const uint32_t keep = in ? 0xFFFFFFFFu : i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
#pragma unroll
                    for (int c = 0; c < BPS; c++) vs[c][i >> 3][(i & 7) >> 1] &= keep;
                } else {
                    const uint32_t keep = in ? 0xFFFFFFFFu : i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
#pragma unroll
                    for (int d = 0; d < NV; d++) vf[d][i >> 1] &= keep;
                }
            }
        }
        if (QUANT) {  // the units of o: the largest scale so far
            us2 top = {0, 0};  // magnitudes compare as integers
            for (int c = 0; c < BPS; c++)
                for (int i = 0; i < 4 * JN; i++) {
                    union { uint32_t u; us2 h; } s;
                    s.u = vs[c][i >> 2][i & 3] & 0x7FFF7FFFu;
                    top = __builtin_elementwise_max(top, s.h);
                }
            const int e = ((int)wave_max((float)max((int)top.x, (int)top.y)) >> 10) - 14;  // every scale < 2^e
            if (e > vexp) {
                const float down = ldexpf(1.0f, vexp - e);
                for (int m = 0; m < TM; m++)
                    for (int d = 0; d < ND; d++) o[m][d] *= down;
                vexp = e;
            }
        }
        const float vunit = ldexpf(1.0f, QUANT ? 14 - vexp : 14);

#pragma unroll
        for (int m = 0; m < TM; m++) {
            float us = unscale[m];
            if (a.softcap > 0.0f) {
                softcap_n<RUN, false>(s[m], us, a.softcap * kLog2e);
                us = 1.0f;
            }
            if (edge)
                for (int i = 0; i < RUN; i++) s[m][i] = kv + i > pos[m] || kv + i < low[m] ? -INFINITY : s[m][i];
            float top = s[m][0];
            for (int i = 1; i < RUN; i++) top = fmaxf(top, s[m][i]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float nm = fmaxf(mx[m], top * us);
            const float down = __builtin_amdgcn_exp2f(mx[m] - nm);
            mx[m] = nm;
            float l = 0.0f;
            if (is_far(nm)) {
                for (int i = 0; i < RUN; i++) s[m][i] *= us;
                us = 1.0f;
            }
            for (int i = 0; i < RUN; i++) {
                s[m][i] = __builtin_amdgcn_exp2f(fmaf(s[m][i], us, -nm));
                l += s[m][i];
            }
            sum[m] = sum[m] * down + l;
            if (__any(down != 1.0f))  // the maximum seldom grows after the first steps
                for (int d = 0; d < ND; d++) o[m][d] *= down;

            if (!QUANT) {
                float w[8];
                for (int i = 0; i < 8; i++) w[i] = s[m][i] * vunit;
                h8 wf[NP];
                split8<NP>(w, wf);
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    H8 v;
                    for (int i = 0; i < 4; i++) v.u[i] = vf[d][i];
                    for (int n = NP - 1; n >= 0; n--) o[m][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v.v, wf[n], o[m][d], 0, 0, 0);
                }
            } else {
                for (int i = 0; i < RUN; i++) s[m][i] *= vunit;
#pragma unroll
                for (int p = 0; p < BPS; p++) {
                    h8 wf[JN][NP];
                    for (int j = 0; j < JN; j++) {
                        float w[8];
                        for (int i = 0; i < 8; i++) {
                            const uint32_t d = vs[p][j][i >> 1];
                            w[i] = i & 1 ? mix_scale<1>(d, s[m][8 * j + i]) : mix_scale<0>(d, s[m][8 * j + i]);
                        }
                        split8<NP>(w, wf[j]);
                    }
#pragma unroll
                    for (int u = 0; u < SUB; u++)
                        for (int h = 0; h < 2; h++)
                            for (int j = 0; j < JN; j++) {
                                const int c = u * BPS + p;
                                const uv& word = vf[TYPE == FLLM_TYPE_Q4_0 ? c : 2 * c + h];
                                const H8 v = codes8<TYPE>(word[2 * j], word[2 * j + 1], h);
                                for (int n = NP - 1; n >= 0; n--)
                                    o[m][2 * c + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v.v, wf[j][n], o[m][2 * c + h], 0, 0, 0);
                            }
                }
            }
        }
        load_v(next);
        pages_at(next + 4 * STEP < it.k1 ? next + 4 * STEP : next);
    }

    // the four waves' results, a row tile at a time
    const float unit = ldexpf(1.0f, QUANT ? vexp - 14 : -14);
    // the tile's partial rows under this kv head: [split][row]
    const int64_t part0 = (int64_t)it.part * a.pg.nkv + (int64_t)kvh * it.nsplit * it.nrows;
    const uint32_t n_part = (uint32_t)(it.nsplit * it.nrows);
    const __amdgpu_buffer_rsrc_t ro = wt_rsrc(a.part_o + part0 * hd, n_part * hd * 4);
    const __amdgpu_buffer_rsrc_t rml = wt_rsrc(a.part_ml + 2 * part0, n_part * 8);
#pragma unroll
    for (int m = 0; m < TM; m++) {
        sum[m] += __shfl_xor(sum[m], 16);
        sum[m] += __shfl_xor(sum[m], 32);
        __syncthreads();  // q, or the tile before, is done with
        if (g == 0 && col < RC) {
            s_m[wave][cq] = mx[m];
            s_l[wave][cq] = sum[m];
        }
#pragma unroll
        for (int d = 0; d < ND; d++)
            if (SUB == 1 || (col < RC * SUB && d / 2 / BPS == sub)) *(f4*)&sm.o[wave][cq][16 * d + 4 * g] = o[m][d] * unit;
        __syncthreads();
        for (int u = threadIdx.x; u < (RC < 16 ? RC : 16) * (HDP / 4); u += 256) {
            const int r = u / (HDP / 4), d = u % (HDP / 4) * 4, row = 16 * m + r;
            if (row >= it.nrows || d >= hd) continue;
            const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
            f4 acc = {0.f, 0.f, 0.f, 0.f};
            float l = 0.0f;
            for (int w = 0; w < 4; w++) {
                const float f = __builtin_amdgcn_exp2f(s_m[w][r] - top);
                l += f * s_l[w][r];
                acc += f * *(const f4*)&sm.o[w][r][d];
            }
            if (it.nsplit == 1) {
                const int tr = it.row0 + row, tok = tr / a.group, head = kvh * a.group + tr % a.group;
                const int64_t at = (int64_t)(it.tok0 + tok) * a.out.ld + (int64_t)head * hd + d;
                const float inv = 1.0f / l;
                store_row4(a.out, at, acc * inv);
            } else {
                const uint32_t pr = (uint32_t)(it.split * it.nrows + row);
                __builtin_amdgcn_raw_buffer_store_b128(acc, ro, (pr * hd + d) * 4, 0, CPOL_SC1);
                if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(f2{top, l}, rml, pr * 8, 0, CPOL_SC1);
            }
        }
    }
    if (it.nsplit == 1) return;

    if (!last_of_tile(a.cnt + part0, it.nsplit, &s_last)) return;
    join_parts<kAttnSplit[0]>(a, it, kvh, ro, rml, sm.w);
}

// ---- many rows -----------------------------------------------------------------------------
// k_attend_many: tiles of up to 128 rows (prompt chunks), bound by the matrix products. Four waves of 32 rows share
// steps of keys whose K and V lie in LDS as halves: one plane where a half holds a value exactly (F16 cache) or the rows
// are 16-bit ones (NP = 1: code times scale, rounded), two planes that hold code times scale exactly (NP = 2); quantised
// values are multiplied by the power of two that brings their step's largest scale to 2^8. S^T is 32 keys by 32
// queries a tile: a lane holds 16 keys of its query, so a row's maximum is one exchange between two lanes.
// Where the halves come from (SRC):
//   SRC_PAGES   an F16 cache's pages, straight to LDS (16 bytes a lane; the LDS image is made by which address a
//               lane loads), two steps deep: the next step arrives while one is multiplied
//   SRC_PARTS   the same from pages shorter than a step: every lane looks up its own
//   SRC_IMAGE   LDS images that k_pages_image made of a quantised cache's pages before, once for all tiles of a
//               sequence, likewise
//   SRC_CODES   a quantised cache's codes, turned into halves by every workgroup: for sequences of few tiles, where
//               writing and reading images costs more than the turning (kImageTiles)
// Measured: 3 prompts of 1500 to 3500 rows behind 500 to 5000, 32 over 8 heads of 128, F16, BF16 rows: 356 GFLOP in 400
// us, 890 TFLOP/s (a large product of halves: 1145), matrix cores busy 43% and the VALU (softmax) 40% of the time at the
// 2.0 GHz that the power limit leaves.
typedef float f16v __attribute__((ext_vector_type(16)));
enum { SRC_PAGES, SRC_PARTS, SRC_IMAGE, SRC_CODES };

constexpr int kManyRows = kAttnTile[kAttnClasses - 1], kManySplit = kAttnSplit[kAttnClasses - 1];

// LDS planes of a step: K [keys][HDP], V [HDP][keys], halves in chunks of 8. Chunk c of a row lies at
// c ^ swizzle(row), so that the 16 lanes that read together (0 to 3, 12 to 15 and 20 to 27, the others of the first 32,
// and so on) cover the banks once.
template <int HDP> __device__ __forceinline__ int k_swizzle(int key) {
    return HDP == 64 ? key >> 1 & 7 : HDP == 128 ? key & 15 : (key & 3) | (key >> 1 & 12);  // 256: k_attend_wide's rows
}
template <int STEP> __device__ __forceinline__ int v_swizzle(int d) {
    return STEP == 64 ? d >> 1 & 7 : ((d >> 3 ^ d >> 2) & 1) << 1 | (d >> 3 & 1);
}
template <int HDP>
__device__ __forceinline__ int k_chunk(int key, int c) {
    return key * (HDP / 8) + (c ^ k_swizzle<HDP>(key));
}
template <int STEP>
__device__ __forceinline__ int v_chunk(int d, int c) {
    return d * (STEP / 8) + (c ^ v_swizzle<STEP>(d));
}

// 8 codes times their scales d (two halves a word, `step` words on for each two codes) times unit, as halves: in one
// plane rounded, or in two exactly, `gap` chunks apart.
template <int KP>
__device__ __forceinline__ void scaled_out(const H8& c, const uint32_t* d, int step, h2 unit, u4* to, int gap) {
    H8 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        union { uint32_t u; h2 h; } s;
        s.u = d[i * step];
        s.h = s.h * unit;
        if (KP == 1) {
            hi.p[i] = c.p[i] * s.h;
        } else {
            const float x = mix_mul<0>(c.u[i], s.u), y = mix_mul<1>(c.u[i], s.u);
            split2(x, y, &hi.p[i], &lo.p[i]);
        }
    }
    to[0] = u4{hi.u[0], hi.u[1], hi.u[2], hi.u[3]};
    if (KP == 2) to[gap] = u4{lo.u[0], lo.u[1], lo.u[2], lo.u[3]};
}

// keys a step: 64, or 32 where q, o and the codes on their way leave too few registers or the planes too little LDS
constexpr int many_step(int hdp, int np) { return hdp > 128 || (hdp == 128 && np == 2) ? 32 : 64; }

// the workgroup's LDS writes (and with DIRECT its loads into LDS) are done, and every wave is here; loads into
// registers stay on their way
template <bool DIRECT>
__device__ __forceinline__ void lds_barrier() {
    if (DIRECT) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void to_lds(const void* from, u4* to) {  // lane l's 16 bytes to to[l]
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// A step's codes of a quantised cache, from the pages into registers and as halves into planes.
template <int TYPE, int HDP, int STEP, int KP, int NT = 256>
struct Codes {
    static constexpr int NB = HDP / 32, PIECES = STEP / 16, CH = STEP * HDP / 8;
    static constexpr int KU = (STEP * NB + NT - 1) / NT;        // (key, block) units a thread
    static constexpr int VROWS = TYPE == FLLM_TYPE_Q4_0 ? HDP / 2 : HDP;
    static constexpr int VU = (VROWS * PIECES + NT - 1) / NT;  // (row, 16 keys) units a thread
    static constexpr int KW = TYPE == FLLM_TYPE_Q8_0 ? 2 : 1;   // 16-byte words of a K unit
    u4 kr[KU][KW], vr[VU], vd[VU][2], ks, vs;  // codes, V's scales, a wave's view of all scales
    uint32_t kd[KU];                           // K's scale of the unit
    int pk, pv[VU], ps;                        // pages of the next step
    float kunit;                               // what K's values are multiplied by
    int vexp;                                  // V's are multiplied by 2^min(8 - vexp, 15)

    __device__ __forceinline__ void pages_at(const int* table, int last_block, int lp, int k0) {
        const auto page_of = [&](int key) { return table[min(key >> lp, last_block)]; };
        pk = page_of(k0 + (int)threadIdx.x % STEP);
#pragma unroll
        for (int i = 0; i < VU; i++) pv[i] = page_of(k0 + 16 * (((int)threadIdx.x + NT * i) / VROWS & (PIECES - 1)));
        ps = page_of(k0 + 8 * ((int)threadIdx.x & (STEP / 8 - 1)));
    }
    __device__ __forceinline__ void load(const PagesView& pg, int kvh, int k0) {
        constexpr int KB = TYPE == FLLM_TYPE_Q8_0 ? 32 : 16;
        const int tid = threadIdx.x, lane = tid & 63, nb = pg.hd >> 5, P = 1 << pg.page_log2;
        const auto cell = [&](int page) { return ((uint64_t)(uint32_t)page * pg.nkv + kvh) * pg.cell; };
        const int key = k0 + tid % STEP;
        const uint8_t* kc = pg.k + cell(pk);
#pragma unroll
        for (int i = 0; i < KU; i++) {
            const int blk = tid / STEP + NT / STEP * i, at = (blk < nb ? blk : 0) * P + (key & (P - 1));
            for (int w = 0; w < KW; w++) kr[i][w] = *(const u4*)(kc + (uint32_t)(at * KB + 16 * w));
            kd[i] = *(const uint16_t*)(kc + pg.scale_off + (uint32_t)(2 * at));
        }
#pragma unroll
        for (int i = 0; i < VU; i++) {
            const int u = tid + NT * i, row = u % VROWS, key16 = k0 + 16 * (u / VROWS & (PIECES - 1));
            const int rows = TYPE == FLLM_TYPE_Q4_0 ? pg.hd / 2 : pg.hd, blk = TYPE == FLLM_TYPE_Q4_0 ? row >> 4 : row >> 5;
            const uint8_t* vc = pg.v + cell(pv[i]);
            vr[i] = *(const u4*)(vc + (uint32_t)((row < rows ? row : 0) * P + (key16 & (P - 1))));
            const uint8_t* sc = vc + pg.scale_off + (uint32_t)(2 * ((blk < nb ? blk : 0) * P + (key16 & (P - 1))));
            vd[i][0] = *(const u4*)sc;
            vd[i][1] = *(const u4*)(sc + 16);
        }
        const int blk = lane / (STEP / 8), at = 2 * ((blk < nb ? blk : 0) * P + ((k0 + 8 * (lane & (STEP / 8 - 1))) & (P - 1)));
        ks = *(const u4*)(pg.k + cell(ps) + pg.scale_off + (uint32_t)at);
        vs = *(const u4*)(pg.v + cell(ps) + pg.scale_off + (uint32_t)at);
    }
    // kunit and vexp from the step's largest scales among the keys [lo, hi) that the sequence has; V scales of zero for
    // the others, which may be anything
    __device__ __forceinline__ void look(int k0, int64_t lo, int64_t hi) {
        const int tid = threadIdx.x, lane = tid & 63;
        us2 tk = {0, 0}, tv = {0, 0};
        const bool outside = k0 < lo || k0 + STEP > hi;
        for (int i = 0; i < 4; i++) {
            union { uint32_t u; us2 h; } x, y;  // magnitudes compare as integers
            x.u = ks[i] & 0x7FFF7FFFu;
            y.u = vs[i] & 0x7FFF7FFFu;
            if (outside) {
                const int64_t key = k0 + 8 * (lane & (STEP / 8 - 1)) + 2 * i;
                const uint32_t keep = (key >= lo && key < hi ? 0xFFFFu : 0u) | (key + 1 >= lo && key + 1 < hi ? 0xFFFF0000u : 0u);
                x.u &= keep;
                y.u &= keep;
            }
            const us2 nan = (us2)(x.h >= us2{0x7C00, 0x7C00});  // no unit: only its own key's scores are lost
            x.h &= ~nan;
            tk = __builtin_elementwise_max(tk, x.h);
            tv = __builtin_elementwise_max(tv, y.h);
        }
        if (outside)
            for (int i = 0; i < VU; i++)
                for (int j = 0; j < 16; j++) {
                    const int64_t key = k0 + 16 * ((tid + NT * i) / VROWS & (PIECES - 1)) + j;
                    vd[i][j >> 3][(j & 7) >> 1] &= key >= lo && key < hi ? 0xFFFFFFFFu : j & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                }
        const int ek = ((int)wave_max((float)max((int)tk.x, (int)tk.y)) >> 10) - 14;  // every scale < 2^ek
        kunit = ldexpf(1.0f, min(8 - ek, 15));
        vexp = ((int)wave_max((float)max((int)tv.x, (int)tv.y)) >> 10) - 14;
    }
    // the codes in registers as halves: K's planes at k, V's at v; V's values for the exponent e >= vexp
    __device__ __forceinline__ void stage(u4* k, u4* v, int e) const {
        const int tid = threadIdx.x;
        const h2 ku = h2{(_Float16)kunit, (_Float16)kunit};
        const _Float16 vf = (_Float16)ldexpf(1.0f, min(8 - e, 15));
        const h2 vu = h2{vf, vf};
#pragma unroll
        for (int i = 0; i < KU; i++) {
            const int key = tid % STEP, blk = tid / STEP + NT / STEP * i;
            if (STEP * NB % NT && blk >= NB) continue;
            const uint32_t d = kd[i] | kd[i] << 16;
            for (int c = 0; c < 4; c++) {
                const u4& w = kr[i][TYPE == FLLM_TYPE_Q8_0 ? c >> 1 & (KW - 1) : 0];
                scaled_out<KP>(codes8<TYPE>(w[2 * (c & 1)], w[2 * (c & 1) + 1], TYPE == FLLM_TYPE_Q8_0 ? 0 : c >> 1), &d, 0, ku,
                               k + k_chunk<HDP>(key, 4 * blk + c), CH);
            }
        }
#pragma unroll
        for (int i = 0; i < VU; i++) {
            const int u = tid + NT * i, row = u % VROWS, piece = u / VROWS;
            if (VROWS * PIECES % NT && piece >= PIECES) continue;
            for (int c = 0; c < 2; c++) {
                const uint32_t d[4] = {vd[i][c].x, vd[i][c].y, vd[i][c].z, vd[i][c].w};
                const int at = TYPE == FLLM_TYPE_Q4_0 ? (row >> 4) * 32 + (row & 15) : row;
                for (int n = 0; n < (TYPE == FLLM_TYPE_Q4_0 ? 2 : 1); n++)
                    scaled_out<KP>(codes8<TYPE>(vr[i][2 * c], vr[i][2 * c + 1], n), d, 1, vu, v + v_chunk<STEP>(at + 16 * n, 2 * piece + c), CH);
            }
        }
    }
};

// A step of an F16 cache's pages to LDS, slot by slot of the LDS image. Where a page holds whole steps (WHOLE) the page
// is the same for all threads; a thread's offsets within the cells never change.
template <int HDP, int STEP, int NT, bool WHOLE>
struct PageLoads {
    static constexpr int CH = STEP * HDP / 8, DL = CH / NT;  // chunks of a plane, loads of one a thread
    uint32_t ko[DL], vo[DL];  // offsets of this thread's slots of K and V in their cells, for position 0 of the step
    int pk[WHOLE ? 1 : DL], pv;  // pages of the next step

    __device__ __forceinline__ void start(const PagesView& pg) {
        const int tid = threadIdx.x, P = 1 << pg.page_log2, nb = pg.hd >> 5;
#pragma unroll
        for (int i = 0; i < DL; i++) {
            const int slot = tid + NT * i, key = slot / (HDP / 8), c = (slot % (HDP / 8)) ^ k_swizzle<HDP>(key);
            ko[i] = (uint32_t)((((c >> 2) < nb ? c >> 2 : 0) * P + (key & (P - 1))) * 64 + (c & 3) * 16);
            const int d = slot / (STEP / 8), b = (slot % (STEP / 8)) ^ v_swizzle<STEP>(d);
            vo[i] = (uint32_t)(((d < pg.hd ? d : 0) * P + (8 * b & (P - 1))) * 2);
        }
    }
    __device__ __forceinline__ void pages_at(const int* table, int last_block, int lp, int k0) {
        const int tid = threadIdx.x;
        if constexpr (WHOLE) {  // the constant address space: a scalar load also beside stores and barriers
            pk[0] = ((const __attribute__((address_space(4))) int*)table)[__builtin_amdgcn_readfirstlane(min(k0 >> lp, last_block))];
        } else {
#pragma unroll
            for (int i = 0; i < DL; i++) pk[i] = table[min((k0 + (tid + NT * i) / (HDP / 8)) >> lp, last_block)];
            // the chunk that this thread's slots of V hold is the same in each: NT slots are a multiple of 16 rows
            pv = table[min((k0 + 8 * ((tid % (STEP / 8)) ^ v_swizzle<STEP>(tid / (STEP / 8)))) >> lp, last_block)];
        }
    }
    __device__ __forceinline__ void load(const PagesView& pg, int kvh, int k0, u4* k, u4* v) const {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const auto cell = [&](int p) { return ((uint64_t)(uint32_t)p * pg.nkv + kvh) * pg.cell; };
        if constexpr (WHOLE) {
            const int at = k0 & ((1 << pg.page_log2) - 1);
            const uint64_t c = cell(pk[0]);
            const uint8_t *kp = pg.k + c + at * 64, *vp = pg.v + c + at * 2;
#pragma unroll
            for (int i = 0; i < DL; i++) to_lds(kp + ko[i], k + NT * i + 64 * wave);
#pragma unroll
            for (int i = 0; i < DL; i++) to_lds(vp + vo[i], v + NT * i + 64 * wave);
        } else {
#pragma unroll
            for (int i = 0; i < DL; i++) to_lds(pg.k + cell(pk[i]) + ko[i], k + NT * i + 64 * wave);
            const uint8_t* vp = pg.v + cell(pv);
#pragma unroll
            for (int i = 0; i < DL; i++) to_lds(vp + vo[i], v + NT * i + 64 * wave);
        }
    }
};

// V of a step in LDS: zeros at the positions outside [lo, hi).
template <int HDP, int STEP, int NT>
__device__ __forceinline__ void zero_outside(u4* v, int k0, int64_t lo, int64_t hi) {
#pragma unroll 1
    for (int u = threadIdx.x; u < HDP * STEP / 8; u += NT) {
        const int d = u / (STEP / 8), c = u % (STEP / 8);
        u4 x = v[v_chunk<STEP>(d, c)];
        for (int j = 0; j < 8; j++) {
            const int64_t key = k0 + 8 * c + j;
            if (key < lo || key >= hi) x[j >> 1] &= j & 1 ? 0x0000FFFFu : 0xFFFF0000u;
        }
        v[v_chunk<STEP>(d, c)] = x;
    }
}

// An image to LDS.
template <int CHUNKS, int NT>
__device__ __forceinline__ void image_to_lds(const u4* image, u4* to) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < CHUNKS / NT; i++) to_lds((const uint8_t*)(image + NT * i) + (uint32_t)threadIdx.x * 16, to + NT * i + 64 * wave);
}

// Images of a quantised cache's steps: [step][kv head] of the planes K, V as they lie in LDS, and of (1 / kunit, vexp).
template <int TYPE, int HDP, int NP>
__global__ __launch_bounds__(256) void k_pages_image(AttnArgsP a, const ImageItem* items) {
    constexpr int STEP = many_step(HDP, NP);
    using C = Codes<TYPE, HDP, STEP, NP>;
    __shared__ u4 planes[2][NP * C::CH];
    const int kvh = blockIdx.x % a.pg.nkv;
    const ImageItem it = items[blockIdx.x / a.pg.nkv];
    const int* table = a.tables + it.table;
    const int last_block = (it.len - 1) >> a.pg.page_log2;
    C c;
    c.pages_at(table, last_block, a.pg.page_log2, it.k0);
    c.load(a.pg, kvh, it.k0);
    for (int i = 0; i < it.n * (kKeyStep / STEP); i++) {
        const int k0 = it.k0 + i * STEP;
        c.look(k0, it.lo, it.len);
        if (i) lds_barrier<false>();  // the image before is copied
        c.stage(planes[0], planes[1], c.vexp);
        const int64_t at = ((int64_t)it.image * (kKeyStep / STEP) + i) * a.pg.nkv + kvh;
        if (threadIdx.x == 0) {
            a.image_units[2 * at] = 1.0f / c.kunit;
            a.image_units[2 * at + 1] = (float)c.vexp;
        }
        c.pages_at(table, last_block, a.pg.page_log2, k0 + STEP);
        c.load(a.pg, kvh, k0 + STEP);
        lds_barrier<false>();
        u4* to = (u4*)a.images + at * (2 * NP * C::CH);
        const u4* from = planes[0];
        for (int u = threadIdx.x; u < 2 * NP * C::CH; u += 256) to[u] = from[u];
    }
}

template <int TYPE, int HDP, int NP, int SRC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_attend_many(AttnArgsP a) {
    constexpr bool QUANT = TYPE != FLLM_TYPE_F16;
    constexpr int KS = HDP / 16, ND = HDP / 32;
    constexpr int KP = QUANT ? NP : 1;                       // planes of K and V
    constexpr int STEP = many_step(HDP, NP), T = STEP / 32;  // keys a step, tiles of 32
    constexpr int CH = STEP * HDP / 8;                       // chunks of 8 halves a plane
    constexpr bool DIRECT = SRC != SRC_CODES;
    // K, V of a step and of the next one: two objects, so that the compiler sees that reads of the one need not wait for
    // loads into the other
    constexpr int WCH = kManySplit * kManyRows / 4;  // the weights of joined parts, in the first one
    __shared__ u4 lds0[2 * KP * CH > WCH ? 2 * KP * CH : WCH], lds1[DIRECT ? 2 * KP * CH : 1];
    __shared__ int s_last;

    const int kvh = blockIdx.x % a.pg.nkv;
    const AttnItem it = a.items[blockIdx.x / a.pg.nkv];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 31, h = lane >> 5;
    const int hd = a.pg.hd, lp = a.pg.page_log2;
    const int* table = a.tables + it.table;
    const int last_block = (it.len - 1) >> lp;
    const int64_t tile_lo = (int64_t)it.pos0 + it.row0 / a.group + 1 - a.window;  // the first key that any row sees

    // ---- the steps on their way; pages of a step are looked up a step before its loads
    Codes<QUANT ? TYPE : (int)FLLM_TYPE_Q8_0, HDP, STEP, KP> codes;  // SRC_CODES
    PageLoads<HDP, STEP, 256, SRC == SRC_PAGES> direct;              // SRC_PAGES, SRC_PARTS
    float ik = 1.0f, ik_next = 1.0f;                                 // quantised: 1 / kunit of this step and the next
    int ev = 0, ev_next = 0;                                         // and vexp
    const auto pages_at = [&](int k0) {
        if (SRC == SRC_CODES) codes.pages_at(table, last_block, lp, k0);
        if (SRC <= SRC_PARTS) direct.pages_at(table, last_block, lp, k0);
    };
    const auto load = [&](int k0, u4* to) {
        if (SRC == SRC_CODES) codes.load(a.pg, kvh, k0);
        if (SRC == SRC_IMAGE) {
            k0 = min(k0, (it.k1 - 1) / STEP * STEP);  // past the item's end: its last step again
            const int64_t at = ((int64_t)it.image * (kKeyStep / STEP) + k0 / STEP) * a.pg.nkv + kvh;
            image_to_lds<2 * KP * CH, 256>((const u4*)a.images + at * (2 * KP * CH), to);
            ik_next = a.image_units[2 * at];
            ev_next = (int)a.image_units[2 * at + 1];
        }
        if (SRC <= SRC_PARTS) direct.load(a.pg, kvh, k0, to, to + KP * CH);
    };
    if (SRC <= SRC_PARTS) direct.start(a.pg);
    pages_at(it.k0);
    load(it.k0, lds0);
    pages_at(it.k0 + STEP);

    // this lane's query
    const int r = 32 * wave + col;
    const bool live = r < it.nrows;
    const int qrow = it.row0 + (live ? r : 0), qtok = qrow / a.group, head = kvh * a.group + qrow % a.group;
    const int pos = live ? it.pos0 + qtok : -1, low = (int)max((int64_t)pos - a.window + 1, (int64_t)INT_MIN);
    float unscale;
    h8 q[KS][NP];
    {
        const int64_t at = (int64_t)(it.tok0 + qtok) * a.q.ld + (int64_t)head * hd;
        float x[KS][8], top = 0.0f;
        if (a.q.type == FLLM_TYPE_F32) {
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const int d = 16 * k + 8 * h;
                const float* p = (const float*)a.q.p + at + (d < hd ? d : 0);
                const f4 u = *(const f4*)p, v = *(const f4*)(p + 4);
                for (int i = 0; i < 4; i++) x[k][i] = u[i], x[k][4 + i] = v[i];
            }
        } else {
            const bool f16 = a.q.type == FLLM_TYPE_F16;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const int d = 16 * k + 8 * h;
                const u4 u = *(const u4*)(a.q.p + 2 * (at + (d < hd ? d : 0)));
                for (int i = 0; i < 4; i++) {
                    union { uint32_t u; h2 h; } c;
                    c.u = u[i];
                    x[k][2 * i] = f16 ? (float)c.h.x : __uint_as_float(u[i] << 16);
                    x[k][2 * i + 1] = f16 ? (float)c.h.y : __uint_as_float(u[i] & 0xFFFF0000u);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < KS; k++)
            for (int i = 0; i < 8; i++) {
                if (!live || 16 * k + 8 * h >= hd) x[k][i] = 0.0f;
                top = fmaxf(top, fabsf(x[k][i]));
            }
        top = fmaxf(top, __shfl_xor(top, 32));
        const int e = row_exponent(top);
        const float up = ldexpf(scale_sign(a.scale), e);
#pragma unroll
        for (int k = 0; k < KS; k++) {
            for (int i = 0; i < 8; i++) x[k][i] *= up;
            split8<NP>(x[k], q[k]);
        }
        unscale = scale_size(a.scale, e, a.softcap);
    }

    f16v o[ND];
    for (int d = 0; d < ND; d++)
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    float mx = kNoScore, sum = 0.0f;
    // keys that every row of the wave sees: [all_lo, all_hi)
    const int w0 = it.row0 + min(32 * wave, it.nrows - 1), w1 = it.row0 + min(32 * wave + 31, it.nrows - 1);
    const int64_t all_hi = it.pos0 + w0 / a.group + 1, all_lo = (int64_t)it.pos0 + w1 / a.group - a.window + 1;

    int vexp = -30;  // quantised: o is in units of 2^-min(8 - vexp, 15), vexp the largest so far
    constexpr float wbits = NP == 2 ? 256.0f : 1.0f;  // weights (up to 2^6) times this: leaves the low halves room
    constexpr bool HALF_SUM = NP == 1 && SRC != SRC_IMAGE;  // an image's weights carry its units, and may vanish in them
    // This lane's operands in a plane: K row krow of a tile, V row col, the chunk 2 k + h of each; chunk bits of k are
    // apart from the row's, so that they are one exclusive or away.
    const int krow = (col & 19) | (col & 4) << 1 | (col & 8) >> 1;
    const int k_at0 = k_chunk<HDP>(krow, h) * 16, v_at0 = v_chunk<STEP>(col, h) * 16;
    const auto step = [&](u4* cur, u4* nxt, int k0) {
        // pages and codes past the item's end are those of its sequence's last page: loaded, never used
        if (SRC == SRC_CODES) {
            codes.look(k0, tile_lo, it.len);
            ik = __builtin_amdgcn_rcpf(codes.kunit);  // a power of two: exact
            ev = max(codes.vexp, vexp);
            if (k0 != it.k0) lds_barrier<false>();  // the step before is read
            codes.stage(cur, cur + KP * CH, ev);
            lds_barrier<false>();
        } else {
            ik = ik_next;
            ev = ev_next;
            lds_barrier<true>();
            if (SRC <= SRC_PARTS && (k0 < tile_lo || k0 + STEP > it.len)) {
                // zeros for what lies outside the sequence, which may be anything
                zero_outside<HDP, STEP, 256>(cur + KP * CH, k0, tile_lo, it.len);
                lds_barrier<false>();
            }
        }
        load(k0 + STEP, nxt);
        pages_at(k0 + 2 * STEP);
        const u4 *kt = cur, *vt = cur + KP * CH;
        int k_at = k_at0, v_at = v_at0;
        asm volatile("" : "+v"(k_at), "+v"(v_at));  // or each address would be kept in a register across the steps

        // S^T = K Q^T: row rho of a 32-key tile is the key with bits 2 and 3 of rho swapped, so that a lane's 8
        // registers 8 s .. are the consecutive keys 16 s + 8 h ..: the second product's operand
        f16v s[T];
#pragma unroll
        for (int t = 0; t < T; t++)
            for (int i = 0; i < 16; i++) s[t][i] = 0.0f;
        union { u4 u; h8 h; } kf[2][T][KP];  // operands of this product and the next
        const auto k_load = [&](int k) {
#pragma unroll
            for (int t = 0; t < T; t++)
                for (int p = 0; p < KP; p++)
                    kf[k & 1][t][p].u = *(const u4*)((const uint8_t*)(kt + p * CH + 32 * t * (HDP / 8)) + (k_at ^ 32 * k));
        };
        k_load(0);
#pragma unroll
        for (int k = 0; k < KS; k++) {
            if (k + 1 < KS) k_load(k + 1);
            __builtin_amdgcn_sched_barrier(0);  // the reads stay ahead of this product
#pragma unroll
            for (int t = 0; t < T; t++) {
                if (KP == 2) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k & 1][t][KP - 1].h, q[k][0], s[t], 0, 0, 0);
                if (NP == 2) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k & 1][t][0].h, q[k][NP - 1], s[t], 0, 0, 0);
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k & 1][t][0].h, q[k][0], s[t], 0, 0, 0);
            }
        }
        float us = unscale;
        if (QUANT) us *= ik;
        if (a.softcap > 0.0f) {
#pragma unroll
            for (int t = 0; t < T; t++) softcap_n<16, true>(s[t], us, a.softcap * kLog2e);
            us = 1.0f;
        }
        const int hide_hi = pos - k0 - 8 * h, hide_lo = low - k0 - 8 * h;
        if (k0 < all_lo || k0 + STEP > all_hi)
#pragma unroll
            for (int t = 0; t < T; t++)
                for (int i = 0; i < 16; i++) {
                    const int key = 32 * t + 16 * (i >> 3) + (i & 7);
                    s[t][i] = key > hide_hi || key < hide_lo ? -INFINITY : s[t][i];
                }
        float top = s[0][0];
#pragma unroll
        for (int t = 0; t < T; t++)
            for (int i = t ? 0 : 1; i < 16; i++) top = fmaxf(top, s[t][i]);
        top = fmaxf(top, __shfl_xor(top, 32)) * us;
        // The weights' reference follows the maximum once one is 2^6 above it: o is seldom multiplied.
        if (__any(top > mx + 6.0f) || (QUANT && ev > vexp)) {
            const float nm = fmaxf(mx, top);
            float down = __builtin_amdgcn_exp2f(mx - nm);
            mx = nm;
            sum *= down;
            if (QUANT && ev > vexp) {
                down *= ldexpf(1.0f, max(vexp, -7) - max(ev, -7));
                vexp = ev;
            }
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= down;
        }
        float wunit = wbits;
        if (SRC == SRC_IMAGE) wunit *= ldexpf(1.0f, max(ev, -7) - max(vexp, -7));  // the step's own units to o's
        if (is_far(mx)) {
#pragma unroll
            for (int t = 0; t < T; t++) s[t] *= us;
            us = 1.0f;
        }
#pragma unroll
        for (int t = 0; t < T; t++)
            for (int i = 0; i < 16; i++) {
                s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], us, -mx));
                if (!HALF_SUM) sum += s[t][i];
            }

        // O^T += V^T P^T
#pragma unroll
        for (int k = 0; k < 2 * T; k++) {
            float w[8];
            for (int i = 0; i < 8; i++) w[i] = s[k >> 1][8 * (k & 1) + i] * wunit;
            h8 wf[NP];
            split8<NP>(w, wf);
            if (HALF_SUM) sum = add_halves(wf[0], sum);
#pragma unroll
            for (int d = 0; d < ND; d++) {
                union { u4 u; h8 h; } vf[KP];
                for (int p = 0; p < KP; p++) vf[p].u = *(const u4*)((const uint8_t*)(vt + p * CH + 32 * d * (STEP / 8)) + (v_at ^ 32 * k));
                if (KP == 2) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[KP - 1].h, wf[0], o[d], 0, 0, 0);
                if (NP == 2) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[0].h, wf[NP - 1], o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[0].h, wf[0], o[d], 0, 0, 0);
            }
        }
    };
    for (int k0 = it.k0;;) {
        step(lds0, DIRECT ? lds1 : lds0, k0);
        if ((k0 += STEP) >= it.k1) break;
        if (!DIRECT) continue;
        step(lds1, lds0, k0);
        if ((k0 += STEP) >= it.k1) break;
    }
    if (DIRECT) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads into LDS that nobody reads

    // results: o in units of 2^-(its scaling)
    sum += __shfl_xor(sum, 32);
    const float unit = ldexpf(1.0f, (QUANT ? -min(8 - vexp, 15) : 0) - (NP == 2 ? 8 : 0));
    if (it.nsplit == 1) {
        const float inv = unit / sum;
        const int64_t at = (int64_t)(it.tok0 + qtok) * a.out.ld + (int64_t)head * hd;
        if (live)
#pragma unroll
            for (int d = 0; d < HDP / 32; d++)
                for (int b = 0; b < 4; b++)
                    if (32 * d < hd) store_row4(a.out, at + 32 * d + 8 * b + 4 * h, f4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]} * inv);
        return;
    }
    const int64_t part0 = (int64_t)it.part * a.pg.nkv + (int64_t)kvh * it.nsplit * it.nrows;
    const uint32_t n_part = (uint32_t)(it.nsplit * it.nrows);
    const __amdgpu_buffer_rsrc_t ro = wt_rsrc(a.part_o + part0 * hd, n_part * hd * 4);
    const __amdgpu_buffer_rsrc_t rml = wt_rsrc(a.part_ml + 2 * part0, n_part * 8);
    if (live) {
        const uint32_t pr = (uint32_t)(it.split * it.nrows + r);
#pragma unroll
        for (int d = 0; d < HDP / 32; d++)
            for (int b = 0; b < 4; b++)
                if (32 * d < hd)
                    __builtin_amdgcn_raw_buffer_store_b128(f4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]} * unit, ro,
                                                           (pr * hd + 32 * d + 8 * b + 4 * h) * 4, 0, CPOL_SC1);
        if (h == 0) __builtin_amdgcn_raw_buffer_store_b64(f2{mx, sum}, rml, pr * 8, 0, CPOL_SC1);
    }
    if (!last_of_tile(a.cnt + part0, it.nsplit, &s_last)) return;
    join_parts<kManySplit>(a, it, kvh, ro, rml, (float*)lds0);
}

// k_attend_wide: the same for heads wider than 128, whose q and o would take all of a 32-row wave's registers: eight
// waves of 16 rows on the 16x16x32 products, two to a SIMD, so that one multiplies while the other reads. S^T tiles and
// operands are k_attend_few's: a lane holds the keys 8 g .. + 8 of a step of 32. Every wave reads all of K and V from
// LDS, which bounds it (4096 cycles a step of 64 KB, a third more than its products). Measured: 2047 rows over a window of 4096, 16 over
// 8 heads of 256, Q8_0, F32 rows (three products of halves for one): 137 GFLOP in 417 us, 35 of them the images; 537 us with
// four waves of 32 rows, whose registers spill.
template <int TYPE, int NP, int SRC>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_attend_wide(AttnArgsP a) {
    constexpr int HDP = 256, NT = 512;
    constexpr bool QUANT = TYPE != FLLM_TYPE_F16;
    constexpr int NB = HDP / 32, ND = HDP / 16;
    constexpr int KP = QUANT ? NP : 1;                       // planes of K and V
    constexpr int STEP = many_step(HDP, NP);                 // keys a step
    static_assert(STEP == 32, "two tiles of 16 keys");
    constexpr int CH = STEP * HDP / 8;                       // chunks of 8 halves a plane
    constexpr bool DIRECT = SRC != SRC_CODES;
    // K, V of a step and of the next one: two objects, so that the compiler sees that reads of the one need not wait for
    // loads into the other
    constexpr int WCH = kManySplit * kManyRows / 4;  // the weights of joined parts, in the first one
    __shared__ u4 lds0[2 * KP * CH > WCH ? 2 * KP * CH : WCH], lds1[DIRECT ? 2 * KP * CH : 1];
    __shared__ int s_last;

    const int kvh = blockIdx.x % a.pg.nkv;
    const AttnItem it = a.items[blockIdx.x / a.pg.nkv];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int hd = a.pg.hd, lp = a.pg.page_log2;
    const int* table = a.tables + it.table;
    const int last_block = (it.len - 1) >> lp;
    const int64_t tile_lo = (int64_t)it.pos0 + it.row0 / a.group + 1 - a.window;  // the first key that any row sees

    // ---- the steps on their way; pages of a step are looked up a step before its loads
    Codes<QUANT ? TYPE : (int)FLLM_TYPE_Q8_0, HDP, STEP, KP, NT> codes;  // SRC_CODES
    PageLoads<HDP, STEP, NT, SRC == SRC_PAGES> direct;               // SRC_PAGES, SRC_PARTS
    float ik = 1.0f, ik_next = 1.0f;                                 // quantised: 1 / kunit of this step and the next
    int ev = 0, ev_next = 0;                                         // and vexp
    const auto pages_at = [&](int k0) {
        if (SRC == SRC_CODES) codes.pages_at(table, last_block, lp, k0);
        if (SRC <= SRC_PARTS) direct.pages_at(table, last_block, lp, k0);
    };
    const auto load = [&](int k0, u4* to) {
        if (SRC == SRC_CODES) codes.load(a.pg, kvh, k0);
        if (SRC == SRC_IMAGE) {
            k0 = min(k0, (it.k1 - 1) / STEP * STEP);  // past the item's end: its last step again
            const int64_t at = ((int64_t)it.image * (kKeyStep / STEP) + k0 / STEP) * a.pg.nkv + kvh;
            image_to_lds<2 * KP * CH, NT>((const u4*)a.images + at * (2 * KP * CH), to);
            ik_next = a.image_units[2 * at];
            ev_next = (int)a.image_units[2 * at + 1];
        }
        if (SRC <= SRC_PARTS) direct.load(a.pg, kvh, k0, to, to + KP * CH);
    };
    if (SRC <= SRC_PARTS) direct.start(a.pg);
    pages_at(it.k0);
    load(it.k0, lds0);
    pages_at(it.k0 + STEP);

    // this lane's query
    const int r = 16 * wave + col;
    const bool live = r < it.nrows;
    const int qrow = it.row0 + (live ? r : 0), qtok = qrow / a.group, head = kvh * a.group + qrow % a.group;
    const int pos = live ? it.pos0 + qtok : -1, low = (int)max((int64_t)pos - a.window + 1, (int64_t)INT_MIN);
    float unscale;
    h8 q[NB][NP];
    {
        const int64_t at = (int64_t)(it.tok0 + qtok) * a.q.ld + (int64_t)head * hd;
        float x[NB][8], top = 0.0f;
        if (a.q.type == FLLM_TYPE_F32) {
#pragma unroll
            for (int c = 0; c < NB; c++) {
                const int d = 32 * c + 8 * g;
                const float* p = (const float*)a.q.p + at + (d < hd ? d : 0);
                const f4 u = *(const f4*)p, v = *(const f4*)(p + 4);
                for (int i = 0; i < 4; i++) x[c][i] = u[i], x[c][4 + i] = v[i];
            }
        } else {
            const bool f16 = a.q.type == FLLM_TYPE_F16;
#pragma unroll
            for (int c = 0; c < NB; c++) {
                const int d = 32 * c + 8 * g;
                const u4 u = *(const u4*)(a.q.p + 2 * (at + (d < hd ? d : 0)));
                for (int i = 0; i < 4; i++) {
                    union { uint32_t u; h2 h; } w;
                    w.u = u[i];
                    x[c][2 * i] = f16 ? (float)w.h.x : __uint_as_float(u[i] << 16);
                    x[c][2 * i + 1] = f16 ? (float)w.h.y : __uint_as_float(u[i] & 0xFFFF0000u);
                }
            }
        }
#pragma unroll
        for (int c = 0; c < NB; c++)
            for (int i = 0; i < 8; i++) {
                if (!live || 32 * c + 8 * g >= hd) x[c][i] = 0.0f;
                top = fmaxf(top, fabsf(x[c][i]));
            }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const int e = row_exponent(top);
        const float up = ldexpf(scale_sign(a.scale), e);
#pragma unroll
        for (int c = 0; c < NB; c++) {
            for (int i = 0; i < 8; i++) x[c][i] *= up;
            split8<NP>(x[c], q[c]);
        }
        unscale = scale_size(a.scale, e, a.softcap);
    }

    f4 o[ND];
    for (int d = 0; d < ND; d++) o[d] = f4{0.f, 0.f, 0.f, 0.f};
    float mx = kNoScore, sum = 0.0f;
    // keys that every row of the wave sees: [all_lo, all_hi)
    const int w0 = it.row0 + min(16 * wave, it.nrows - 1), w1 = it.row0 + min(16 * wave + 15, it.nrows - 1);
    const int64_t all_hi = it.pos0 + w0 / a.group + 1, all_lo = (int64_t)it.pos0 + w1 / a.group - a.window + 1;

    int vexp = -30;  // quantised: o is in units of 2^-min(8 - vexp, 15), vexp the largest so far
    constexpr float wbits = NP == 2 ? 256.0f : 1.0f;  // weights (up to 2^6) times this: leaves the low halves room
    // this lane's operands in a plane: K row 8 (col >> 2) + (col & 3) of tile 0, the chunk 4 c + g; V row col, the chunk g
    const int k_at0 = k_chunk<HDP>(8 * (col >> 2) + (col & 3), g) * 16, v_at0 = v_chunk<STEP>(col, g) * 16;
    const auto step = [&](u4* cur, u4* nxt, int k0) {
        // pages and codes past the item's end are those of its sequence's last page: loaded, never used
        if (SRC == SRC_CODES) {
            codes.look(k0, tile_lo, it.len);
            ik = __builtin_amdgcn_rcpf(codes.kunit);  // a power of two: exact
            ev = max(codes.vexp, vexp);
            if (k0 != it.k0) lds_barrier<false>();  // the step before is read
            codes.stage(cur, cur + KP * CH, ev);
            lds_barrier<false>();
        } else {
            ik = ik_next;
            ev = ev_next;
            lds_barrier<true>();
            if (SRC <= SRC_PARTS && (k0 < tile_lo || k0 + STEP > it.len)) {
                // zeros for what lies outside the sequence, which may be anything
                zero_outside<HDP, STEP, NT>(cur + KP * CH, k0, tile_lo, it.len);
                lds_barrier<false>();
            }
        }
        load(k0 + STEP, nxt);
        pages_at(k0 + 2 * STEP);
        const u4 *kt = cur, *vt = cur + KP * CH;
        int k_at = k_at0, v_at = v_at0;
        asm volatile("" : "+v"(k_at), "+v"(v_at));  // or each address would be kept in a register across the steps

        // S^T = K Q^T: row rho of tile t is key 8 (rho >> 2) + 4 t + (rho & 3); high and low products apart, so that there
        // are four chains of them
        f4 hi[2], lo[2];
#pragma unroll
        for (int t = 0; t < 2; t++) hi[t] = lo[t] = f4{0.f, 0.f, 0.f, 0.f};
        union { u4 u; h8 h; } kf[2][2][KP];  // operands of this product and the next
        const auto k_load = [&](int c) {
#pragma unroll
            for (int t = 0; t < 2; t++)
                for (int p = 0; p < KP; p++)
                    kf[c & 1][t][p].u = *(const u4*)((const uint8_t*)(kt + p * CH + 4 * t * (HDP / 8)) + (k_at ^ 64 * c));
        };
        k_load(0);
#pragma unroll
        for (int c = 0; c < NB; c++) {
            if (c + 1 < NB) k_load(c + 1);
            __builtin_amdgcn_sched_barrier(0);  // the reads stay ahead of this product
#pragma unroll
            for (int t = 0; t < 2; t++) {
                hi[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[c & 1][t][0].h, q[c][0], hi[t], 0, 0, 0);
                if (NP == 2) lo[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[c & 1][t][0].h, q[c][NP - 1], lo[t], 0, 0, 0);
                if (KP == 2) lo[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[c & 1][t][KP - 1].h, q[c][0], lo[t], 0, 0, 0);
            }
        }
        float s[8];
        for (int i = 0; i < 8; i++) s[i] = NP == 2 ? hi[i >> 2][i & 3] + lo[i >> 2][i & 3] : hi[i >> 2][i & 3];
        float us = unscale;
        if (QUANT) us *= ik;
        if (a.softcap > 0.0f) {
            softcap_n<8, true>(s, us, a.softcap * kLog2e);
            us = 1.0f;
        }
        const int hide_hi = pos - k0 - 8 * g, hide_lo = low - k0 - 8 * g;
        if (k0 < all_lo || k0 + STEP > all_hi)
            for (int i = 0; i < 8; i++) {
                s[i] = i > hide_hi || i < hide_lo ? -INFINITY : s[i];
            }
        float top = s[0];
        for (int i = 1; i < 8; i++) top = fmaxf(top, s[i]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32)) * us;
        // The weights' reference follows the maximum once one is 2^6 above it: o is seldom multiplied.
        if (__any(top > mx + 6.0f) || (QUANT && ev > vexp)) {
            const float nm = fmaxf(mx, top);
            float down = __builtin_amdgcn_exp2f(mx - nm);
            mx = nm;
            sum *= down;
            if (QUANT && ev > vexp) {
                down *= ldexpf(1.0f, max(vexp, -7) - max(ev, -7));
                vexp = ev;
            }
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= down;
        }
        float wunit = wbits;
        if (SRC == SRC_IMAGE) wunit *= ldexpf(1.0f, max(ev, -7) - max(vexp, -7));  // the step's own units to o's
        float w[8], l = 0.0f;
        if (is_far(mx)) {
            for (int i = 0; i < 8; i++) s[i] *= us;
            us = 1.0f;
        }
        for (int i = 0; i < 8; i++) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], us, -mx));
            l += s[i];
            w[i] = s[i] * wunit;
        }
        sum += l;
        h8 wf[NP];
        split8<NP>(w, wf);

        // O^T += V^T P^T
#pragma unroll
        for (int d = 0; d < ND; d++) {
            union { u4 u; h8 h; } vf[KP];
            for (int p = 0; p < KP; p++) vf[p].u = *(const u4*)((const uint8_t*)(vt + p * CH + 16 * d * (STEP / 8)) + v_at);
            if (KP == 2) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[KP - 1].h, wf[0], o[d], 0, 0, 0);
            if (NP == 2) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[0].h, wf[NP - 1], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[0].h, wf[0], o[d], 0, 0, 0);
        }
    };
    for (int k0 = it.k0;;) {
        step(lds0, DIRECT ? lds1 : lds0, k0);
        if ((k0 += STEP) >= it.k1) break;
        if (!DIRECT) continue;
        step(lds1, lds0, k0);
        if ((k0 += STEP) >= it.k1) break;
    }
    if (DIRECT) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads into LDS that nobody reads

    // results: o in units of 2^-(its scaling)
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    const float unit = ldexpf(1.0f, (QUANT ? -min(8 - vexp, 15) : 0) - (NP == 2 ? 8 : 0));
    if (it.nsplit == 1) {
        const float inv = unit / sum;
        const int64_t at = (int64_t)(it.tok0 + qtok) * a.out.ld + (int64_t)head * hd;
        if (live)
#pragma unroll
            for (int d = 0; d < ND; d++)
                if (16 * d < hd) store_row4(a.out, at + 16 * d + 4 * g, o[d] * inv);
        return;
    }
    const int64_t part0 = (int64_t)it.part * a.pg.nkv + (int64_t)kvh * it.nsplit * it.nrows;
    const uint32_t n_part = (uint32_t)(it.nsplit * it.nrows);
    const __amdgpu_buffer_rsrc_t ro = wt_rsrc(a.part_o + part0 * hd, n_part * hd * 4);
    const __amdgpu_buffer_rsrc_t rml = wt_rsrc(a.part_ml + 2 * part0, n_part * 8);
    if (live) {
        const uint32_t pr = (uint32_t)(it.split * it.nrows + r);
#pragma unroll
        for (int d = 0; d < ND; d++)
            if (16 * d < hd) __builtin_amdgcn_raw_buffer_store_b128(o[d] * unit, ro, (pr * hd + 16 * d + 4 * g) * 4, 0, CPOL_SC1);
        if (g == 0) __builtin_amdgcn_raw_buffer_store_b64(f2{mx, sum}, rml, pr * 8, 0, CPOL_SC1);
    }
    if (!last_of_tile(a.cnt + part0, it.nsplit, &s_last)) return;
    join_parts<kManySplit, NT>(a, it, kvh, ro, rml, (float*)lds0);
}

inline AttnArgsP attend_args(const PagesView& pg, const BatchView& b, const AttnWork& w, const RowsView& q, const RowsView& out,
                             float scale, float softcap) {
    return AttnArgsP{pg, b.tables, nullptr, b.n_heads / pg.nkv, b.window, q, out, scale, softcap,
                     w.part, w.part + w.part_rows * pg.nkv * pg.hd, w.cnt, w.images, w.image_units};
}

template <int TYPE, int HDP, int NP>
hipError_t launch_items(AttnArgsP a, const AttnWork& w, hipStream_t st) {
    constexpr bool QUANT = TYPE != FLLM_TYPE_F16;
    const auto grid = [&](int c) { return dim3((unsigned)w.n[c] * (unsigned)a.pg.nkv); };
    // the long-running tiles first
    for (int c = kAttnClasses - 1; c >= 0; c--) {
        if (w.n[c] == 0) continue;
        a.items = w.items[c];
        if (c == kAttnImage) {
            if constexpr (QUANT) {
                hipLaunchKernelGGL((k_pages_image<TYPE, HDP, NP>), dim3((unsigned)w.n_image_items * (unsigned)a.pg.nkv), dim3(256), 0, st, a, w.image_items);
                const hipError_t e = hipGetLastError();
                if (e != hipSuccess) return e;
                if constexpr (HDP > 128) hipLaunchKernelGGL((k_attend_wide<TYPE, NP, SRC_IMAGE>), grid(c), dim3(512), 0, st, a);
                else hipLaunchKernelGGL((k_attend_many<TYPE, HDP, NP, SRC_IMAGE>), grid(c), dim3(256), 0, st, a);
            }
        } else if (c == kAttnMany) {
            const bool whole = 1 << a.pg.page_log2 >= many_step(HDP, NP);
            const auto go = [&](auto src) {
                constexpr int SRC = decltype(src)::value;
                if constexpr (HDP > 128) hipLaunchKernelGGL((k_attend_wide<TYPE, NP, SRC>), grid(c), dim3(512), 0, st, a);
                else hipLaunchKernelGGL((k_attend_many<TYPE, HDP, NP, SRC>), grid(c), dim3(256), 0, st, a);
            };
            if constexpr (QUANT) go(std::integral_constant<int, SRC_CODES>());
            else if (whole) go(std::integral_constant<int, SRC_PAGES>());
            else go(std::integral_constant<int, SRC_PARTS>());
        } else if (c == 3) {
            if constexpr (!QUANT && HDP <= 128) hipLaunchKernelGGL((k_attend_few<TYPE, HDP, NP, 2, 16>), grid(c), dim3(256), 0, st, a);
        } else if (c == 2) {
            hipLaunchKernelGGL((k_attend_few<TYPE, HDP, NP, 1, 16>), grid(c), dim3(256), 0, st, a);
        } else {
            if constexpr (QUANT) {
                if (c == 1) hipLaunchKernelGGL((k_attend_few<TYPE, HDP, NP, 1, 8>), grid(c), dim3(256), 0, st, a);
                else hipLaunchKernelGGL((k_attend_few<TYPE, HDP, NP, 1, 4>), grid(c), dim3(256), 0, st, a);
            }
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int TYPE, int NP>
hipError_t launch_items_hd(const AttnArgsP& a, const AttnWork& w, hipStream_t st) {
    if (a.pg.hd <= 64) return launch_items<TYPE, 64, NP>(a, w, st);
    if (a.pg.hd <= 128) return launch_items<TYPE, 128, NP>(a, w, st);
    return launch_items<TYPE, 256, NP>(a, w, st);
}

template <int TYPE>
hipError_t launch_items_of(const AttnArgsP& a, const AttnWork& w, hipStream_t st) {
    // 16-bit rows: 11-bit factors lose less than their outputs' rounding
    return a.q.type == FLLM_TYPE_F32 || a.out.type == FLLM_TYPE_F32 ? launch_items_hd<TYPE, 2>(a, w, st)
                                                                    : launch_items_hd<TYPE, 1>(a, w, st);
}

}  // namespace
}  // namespace fllm
