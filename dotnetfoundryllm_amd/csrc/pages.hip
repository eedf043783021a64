// pages.hip — rows into and out of the pages of the paged K/V cache.
//
// A workgroup takes the positions of one page that the call covers, for one kv head and one of K and V: up to
// page_size rows of head_dim. Both kernels are bound by memory traffic for many rows and by the launch's chain of
// loads (lengths, page, rows) for few. On the dense side a lane moves 16 bytes (F32 rows: 4 elements, a wave 1 KiB
// of consecutive ones). K keeps the rows' direction, so its codes go straight to their place. V lies with the
// positions along the row (what the attention's second product reads): its codes pass through LDS as [position][row],
// and a thread turns 4 rows by 16 positions in registers (byte permutes), so that the pages are read and written 16
// bytes at a time too. Measured: 8 sequences of 3000 to 16000 positions, 8 heads of 256, Q8_0 to F16 rows: 825 MB in
// 202 us (4.1 TB/s; a 1 GiB copy reaches 5.1); four prompts of 900 to 4000 rows, 4 heads of 128, F32 to Q4_0 and back:
// 73 MB in 21.8 us, two launches; one row of 64 sequences in and out: 8.9 us, of which two empty launches are 7.4.
#include "pages.hpp"

namespace fllm {

namespace {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

struct Tile {
    int off, n;     // first position in the page, number of positions
    int64_t row;    // their first row in the dense matrix
    uint64_t cell;  // the cell's offset
};

// Tile `at` of the new tokens, one load away, or of all positions: page `at` of the sequences' pages, whose sequence a wave
// finds with one load for up to 64 of them (202 us of the case at grid_of; 212 by halving).
__device__ __forceinline__ Tile tile_of(const PagesView& pg, const BatchView& b, bool new_only, int at, int head) {
    Tile t;
    int page;
    if (new_only) {
        const int4 q = b.new_tiles[at];
        t.off = q.x;
        t.n = q.y;
        t.row = q.z;
        page = q.w;
    } else {
        int s = 0, start = 0;  // the last sequence whose pages start at `at` or before, and where they do
        for (int n = b.n_seqs; n > 1;) {
            const int step = (n + 63) >> 6, i = (int)(threadIdx.x & 63) * step;
            const int f = b.first[s + (i < n ? i : 0)], k = __builtin_popcountll(__ballot(i < n && f <= at)) - 1;
            start = __builtin_amdgcn_readlane(f, k);
            s += k * step;
            n = min(step, n - k * step);
        }
        const int4 q = b.seqs[s];
        const int pos = (at - start) << pg.page_log2;
        t.off = 0;
        t.n = min(q.z - pos, 1 << pg.page_log2);
        t.row = (int64_t)q.w + pos;
        page = b.tables[at];
    }
    t.cell = ((uint64_t)(uint32_t)page * pg.nkv + head) * pg.cell;
    return t;
}

__device__ __forceinline__ uint32_t half_bits(float f) {
    const _Float16 h = (_Float16)f;
    uint16_t u;
    __builtin_memcpy(&u, &h, 2);
    return u;
}
__device__ __forceinline__ float half_float(uint32_t u) {
    const uint16_t b = (uint16_t)u;
    _Float16 h;
    __builtin_memcpy(&h, &b, 2);
    return (float)h;
}

// 8 elements of a row
__device__ __forceinline__ void load8(const RowsView& r, int64_t i, float x[8]) {
    if (r.type == FLLM_TYPE_F32) {
        const float4 a = *(const float4*)(r.p + 4 * i), b = *(const float4*)(r.p + 4 * i + 16);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        return;
    }
    const uint4 u = *(const uint4*)(r.p + 2 * i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    for (int e = 0; e < 4; e++) {
        x[2 * e] = r.type == FLLM_TYPE_F16 ? half_float(w[e] & 0xFFFFu) : __uint_as_float(w[e] << 16);
        x[2 * e + 1] = r.type == FLLM_TYPE_F16 ? half_float(w[e] >> 16) : __uint_as_float(w[e] & 0xFFFF0000u);
    }
}

// The integer nearest to x / d (ties to even), clamped: the rounded product with the reciprocal is at
// most one off, and the remainder x - c d (exact in one fma: c d has 19 bits) says in which
// direction. A float32 division would round a quotient next to a tie onto it.
__device__ __forceinline__ int code_of(float x, float d, float inv, float half, int lo, int hi) {
    const float c = fminf(fmaxf(rintf(x * inv), -300.0f), 300.0f);
    const float r = fmaf(-c, d, x);
    const float s = d < 0.0f ? -r : r;  // remainder in units of |d|
    const bool odd = (int)c & 1;
    float q = c;
    if (s > half || (s == half && odd)) q += 1.0f;
    else if (s < -half || (s == -half && odd)) q -= 1.0f;
    return (int)fminf(fmaxf(q, (float)lo), (float)hi);
}

// within a quad of lanes (DPP): the value of the lane whose number differs in bit 0, in bit 1
__device__ __forceinline__ uint32_t quad_xor1(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true); }
__device__ __forceinline__ uint32_t quad_xor2(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true); }

// The scale of a block of 32 over its 4 lanes, 8 elements each: its bits in half precision.
template <int TYPE>
__device__ __forceinline__ uint32_t block_scale(const float x[8], int e) {
    uint32_t top = 0;  // magnitudes compare as integers; a NaN's is above all
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = max(top, quad_xor1(top));
    top = max(top, quad_xor2(top));
    if (top >= 0x7F800000u) return 0x7E00u;  // not finite: a NaN scale
    float d;
    if (TYPE == FLLM_TYPE_Q8_0) {
        d = __uint_as_float(top) / 127.0f;
    } else {
        uint32_t at = ~0u;  // the first element of that magnitude, its sign in the low bit
        for (int i = 7; i >= 0; i--)
            if ((__float_as_uint(x[i]) & 0x7FFFFFFFu) == top) at = (uint32_t)(8 * e + i) << 1 | __float_as_uint(x[i]) >> 31;
        at = min(at, quad_xor1(at));
        at = min(at, quad_xor2(at));
        d = __uint_as_float(top) * (at & 1u ? 0.125f : -0.125f);
    }
    const uint32_t h = half_bits(d);
    return (h & 0x7FFFu) == 0x7C00u ? (h & 0x8000u) | 0x7BFFu : h;
}

// 4 words of 4 bytes each as their transpose
__device__ __forceinline__ void turn4(const uint32_t w[4], uint32_t o[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    o[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    o[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    o[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    o[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// V's rows of a cell (two elements a byte row in Q4_0), bytes of one position in a row
template <int TYPE> __device__ __host__ constexpr int v_rows(int hd) { return TYPE == FLLM_TYPE_Q4_0 ? hd / 2 : hd; }
template <int TYPE> __device__ __host__ constexpr int v_bytes() { return TYPE == FLLM_TYPE_F16 ? 2 : 1; }
template <int TYPE> __device__ __host__ constexpr int lds_pitch(int hd) { return v_rows<TYPE>(hd) * v_bytes<TYPE>() + 16; }

template <int TYPE>
__global__ __launch_bounds__(256) void k_pages_append(PagesView pg, BatchView b, int nb_log2, RowsView rk, RowsView rv) {
    extern __shared__ __align__(16) uint8_t turned[];  // V's codes, [position][row]
    const int head = blockIdx.x >> 1, kind = blockIdx.x & 1;
    const int P = 1 << pg.page_log2, nb = pg.hd >> 5;
    const RowsView& src = kind ? rv : rk;
    const int pitch = lds_pitch<TYPE>(pg.hd);
    for (int at = blockIdx.y; at < b.n_new_tiles; at += gridDim.y) {
        const Tile t = tile_of(pg, b, true, at, head);
        uint8_t* cell = (kind ? pg.v : pg.k) + t.cell;
        const int e = threadIdx.x & 3;
        for (int u = threadIdx.x >> 2; u < t.n << nb_log2; u += blockDim.x >> 2) {
            const int i = u >> nb_log2, blk = u & ((1 << nb_log2) - 1), pos = t.off + i;
            if (blk >= nb) continue;
            float x[8];
            load8(src, (t.row + i) * src.ld + head * pg.hd + blk * 32 + 8 * e, x);
            uint4 c;
            if (TYPE == FLLM_TYPE_F16) {
                c = make_uint4(half_bits(x[0]) | half_bits(x[1]) << 16, half_bits(x[2]) | half_bits(x[3]) << 16,
                               half_bits(x[4]) | half_bits(x[5]) << 16, half_bits(x[6]) | half_bits(x[7]) << 16);
            } else {
                const uint32_t h = block_scale<TYPE>(x, e);
                const float d = half_float(h);
                const bool live = d != 0.0f && d == d;
                const float inv = live ? 1.0f / d : 0.0f, half = 0.5f * fabsf(d);
                uint32_t w[2] = {0, 0};
                for (int j = 0; j < 8; j++) {
                    const int q = !live ? 0 : TYPE == FLLM_TYPE_Q8_0 ? code_of(x[j], d, inv, half, -127, 127)
                                                                     : code_of(x[j], d, inv, half, -8, 7);
                    w[j >> 2] |= (TYPE == FLLM_TYPE_Q8_0 ? (uint32_t)q & 0xFFu : (uint32_t)(q + 8)) << 8 * (j & 3);
                }
                if (e == 0) *(uint16_t*)(cell + pg.scale_off + 2 * (blk * P + pos)) = (uint16_t)h;
                if (TYPE == FLLM_TYPE_Q4_0) {  // the upper 16 elements' codes join the lower ones' bytes
                    w[0] |= quad_xor2(w[0]) << 4;
                    w[1] |= quad_xor2(w[1]) << 4;
                    if (e >= 2) continue;
                }
                c.x = w[0], c.y = w[1];
            }
            constexpr int PER = TYPE == FLLM_TYPE_F16 ? 64 : TYPE == FLLM_TYPE_Q8_0 ? 32 : 16;  // bytes of a block
            uint8_t* to = kind ? turned + pos * pitch + blk * PER : cell + (blk * P + pos) * PER;
            if (TYPE == FLLM_TYPE_F16) *(uint4*)(to + 16 * e) = c;
            else *(uint2*)(to + 8 * e) = make_uint2(c.x, c.y);
        }
        if (kind == 0) continue;
        __syncthreads();
        // 4 rows by 16 bytes of positions a thread
        constexpr int VB = v_bytes<TYPE>(), RUN = 16 / VB;
        const int pieces = P / RUN, units = v_rows<TYPE>(pg.hd) / 4 * pieces, lo0 = t.off / RUN;
        const int held = (t.off + t.n - 1) / RUN - lo0 + 1;  // pieces with new positions
        for (int u = threadIdx.x; u < units / pieces * held; u += blockDim.x) {
            const int row = u / held * 4, piece = lo0 + u % held;
            const uint8_t* from = turned + piece * RUN * pitch + row * VB;
            uint8_t* to = cell + (row * P + piece * RUN) * VB;
            if (piece * RUN >= t.off && (piece + 1) * RUN <= t.off + t.n) {
                uint32_t o[4][4];
                if (TYPE == FLLM_TYPE_F16) {
                    for (int j = 0; j < 4; j++) {
                        const uint2 a = *(const uint2*)(from + 2 * j * pitch), c = *(const uint2*)(from + (2 * j + 1) * pitch);
                        o[0][j] = __builtin_amdgcn_perm(c.x, a.x, 0x05040100u);
                        o[1][j] = __builtin_amdgcn_perm(c.x, a.x, 0x07060302u);
                        o[2][j] = __builtin_amdgcn_perm(c.y, a.y, 0x05040100u);
                        o[3][j] = __builtin_amdgcn_perm(c.y, a.y, 0x07060302u);
                    }
                } else {
                    for (int j = 0; j < 4; j++) {
                        uint32_t w[4], q[4];
                        for (int k = 0; k < 4; k++) w[k] = *(const uint32_t*)(from + (4 * j + k) * pitch);
                        turn4(w, q);
                        for (int k = 0; k < 4; k++) o[k][j] = q[k];
                    }
                }
                for (int k = 0; k < 4; k++) *(uint4*)(to + k * P * VB) = make_uint4(o[k][0], o[k][1], o[k][2], o[k][3]);
            } else {
                for (int i = max(0, t.off - piece * RUN); i < min(RUN, t.off + t.n - piece * RUN); i++)
                    for (int k = 0; k < 4; k++) {
                        if (TYPE == FLLM_TYPE_F16) ((uint16_t*)to)[k * P + i] = *(const uint16_t*)(from + i * pitch + 2 * k);
                        else to[k * P + i] = from[i * pitch + k];
                    }
            }
        }
        __syncthreads();
    }
}

// EL: elements a lane writes, 16 bytes of the dense rows
template <int TYPE, int EL>
__global__ __launch_bounds__(256) void k_pages_read(PagesView pg, BatchView b, bool new_only, int el_log2, RowsView rk, RowsView rv) {
    extern __shared__ __align__(16) uint8_t turned[];
    const int head = blockIdx.x >> 1, kind = blockIdx.x & 1;
    const RowsView& dst = kind ? rv : rk;
    if (!dst.p) return;
    const int P = 1 << pg.page_log2;
    const int pitch = lds_pitch<TYPE>(pg.hd);
    constexpr int VB = v_bytes<TYPE>(), RUN = 16 / VB;
    constexpr int PER = TYPE == FLLM_TYPE_F16 ? 64 : TYPE == FLLM_TYPE_Q8_0 ? 32 : 16;
    const int tiles = new_only ? b.n_new_tiles : b.n_blocks;
    for (int at = blockIdx.y; at < tiles; at += gridDim.y) {
        const Tile t = tile_of(pg, b, new_only, at, head);
        const uint8_t* cell = (kind ? pg.v : pg.k) + t.cell;
        if (kind) {
            const int lo0 = t.off / RUN, held = (t.off + t.n - 1) / RUN - lo0 + 1;
            for (int u = threadIdx.x; u < v_rows<TYPE>(pg.hd) / 4 * held; u += blockDim.x) {
                const int row = u / held * 4, piece = lo0 + u % held;
                const uint8_t* from = cell + (row * P + piece * RUN) * VB;
                uint8_t* to = turned + piece * RUN * pitch + row * VB;
                uint32_t w[4][4];
                for (int k = 0; k < 4; k++) {
                    const uint4 v = *(const uint4*)(from + k * P * VB);
                    w[k][0] = v.x, w[k][1] = v.y, w[k][2] = v.z, w[k][3] = v.w;
                }
                for (int j = 0; j < 4; j++) {
                    if (TYPE == FLLM_TYPE_F16) {
                        *(uint2*)(to + 2 * j * pitch) = make_uint2(__builtin_amdgcn_perm(w[1][j], w[0][j], 0x05040100u),
                                                                   __builtin_amdgcn_perm(w[3][j], w[2][j], 0x05040100u));
                        *(uint2*)(to + (2 * j + 1) * pitch) = make_uint2(__builtin_amdgcn_perm(w[1][j], w[0][j], 0x07060302u),
                                                                         __builtin_amdgcn_perm(w[3][j], w[2][j], 0x07060302u));
                    } else {
                        const uint32_t in[4] = {w[0][j], w[1][j], w[2][j], w[3][j]};
                        uint32_t q[4];
                        turn4(in, q);
                        for (int k = 0; k < 4; k++) *(uint32_t*)(to + (4 * j + k) * pitch) = q[k];
                    }
                }
            }
            __syncthreads();
        }
        // a lane per EL elements, 2^el_log2 lanes (some idle) a row; 4 of them on their way
        const int live = pg.hd / EL, all = t.n << el_log2;
        for (int u0 = threadIdx.x; u0 < all; u0 += 4 * blockDim.x) {
            uint32_t w[4][EL / 2];
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int u = u0 + k * (int)blockDim.x, lane = u & ((1 << el_log2) - 1);
                if (u >= all || lane >= live) continue;
                const int pos = t.off + (u >> el_log2), d = lane * EL, blk = d >> 5, in = d & 31;
                const uint8_t* row = kind ? turned + pos * pitch + blk * PER : cell + (blk * P + pos) * PER;
                if (TYPE == FLLM_TYPE_F16) {
                    for (int j = 0; j < EL / 2; j += 2) {
                        const uint2 v = *(const uint2*)(row + 2 * in + 4 * j);
                        w[k][j] = v.x, w[k][j + 1] = v.y;
                    }
                } else {
                    h[k] = *(const uint16_t*)(cell + pg.scale_off + 2 * (blk * P + pos));
                    for (int j = 0; j < EL / 4; j++) w[k][j] = *(const uint32_t*)(row + (in & (PER - 1)) + 4 * j);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int u = u0 + k * (int)blockDim.x, lane = u & ((1 << el_log2) - 1);
                if (u >= all || lane >= live) continue;
                float x[EL];
                if (TYPE == FLLM_TYPE_F16) {
                    for (int j = 0; j < EL / 2; j++) {
                        x[2 * j] = half_float(w[k][j] & 0xFFFFu);
                        x[2 * j + 1] = half_float(w[k][j] >> 16);
                    }
                } else {
                    const float d = half_float(h[k]);
                    const int up = TYPE == FLLM_TYPE_Q4_0 && (lane * EL & 16) ? 4 : 0;
                    for (int j = 0; j < EL; j++) {
                        const uint32_t c = w[k][j >> 2] >> 8 * (j & 3);
                        const int q = TYPE == FLLM_TYPE_Q8_0 ? (int)(int8_t)(c & 0xFFu) : (int)(c >> up & 15u) - 8;
                        x[j] = (float)q * d;
                    }
                }
                uint8_t* to = dst.p + ((t.row + (u >> el_log2)) * dst.ld + head * pg.hd + lane * EL) * (16 / EL);
                // past the caches (the rows are not read here again): 204 us in place of 217 of the case at grid_of
                if (EL == 4) {
                    __builtin_nontemporal_store(f4v{x[0], x[1], x[2], x[3]}, (f4v*)to);
                } else {
                    uint32_t o[EL];
                    for (int j = 0; j < EL; j++) o[j] = dst.type == FLLM_TYPE_F16 ? half_bits(x[j]) : bf16_round(x[j]);
                    __builtin_nontemporal_store(u4v{o[0] | o[1] << 16, o[2] | o[3] << 16, o[EL - 4] | o[EL - 3] << 16, o[EL - 2] | o[EL - 1] << 16}, (u4v*)to);
                }
            }
        }
        __syncthreads();
    }
}

int log2_up(int n) {
    int k = 0;
    while (1 << k < n) k++;
    return k;
}

// A tile of few rows has little work for 256 threads: one wave starts sooner and leaves the CU to others (64 sequences of 8
// heads of 128, Q8_0, in and out, in us with 256 and 64 threads: 1 row 9.5 and 8.7, 4 rows 16.3 and 13.3, 8 rows 20.5
// and 19.1).
int threads_for(const PagesView& pg, int rows) { return rows * (pg.hd >> 5) <= 32 ? 64 : 256; }

// The heads of a page follow each other, so that what lies side by side in the dense rows moves at the same time
// (8 sequences of 3000 to 16000 positions, 8 heads of 256, Q8_0 to F16: 249 us with the pages of a head in a row, then
// 217). The second dimension ends at 65535: the kernels go on from there.
dim3 grid_of(const PagesView& pg, int tiles) { return dim3(2 * pg.nkv, tiles < 65535 ? tiles : 65535); }

template <int TYPE>
hipError_t append(const PagesView& pg, const BatchView& b, const RowsView& k, const RowsView& v, hipStream_t st) {
    const dim3 grid = grid_of(pg, b.n_new_tiles);
    const size_t lds = (size_t)lds_pitch<TYPE>(pg.hd) << pg.page_log2;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)k_pages_append<TYPE>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(k_pages_append<TYPE>, grid, dim3(threads_for(pg, b.max_new)), lds, st, pg, b, log2_up(pg.hd / 32), k, v);
    return hipGetLastError();
}

template <int TYPE, int EL>
hipError_t read(const PagesView& pg, const BatchView& b, bool new_only, const RowsView& k, const RowsView& v, hipStream_t st) {
    const dim3 grid = grid_of(pg, new_only ? b.n_new_tiles : b.n_blocks);
    const size_t lds = (size_t)lds_pitch<TYPE>(pg.hd) << pg.page_log2;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)k_pages_read<TYPE, EL>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    const int rows = new_only ? b.max_new : 1 << pg.page_log2;
    hipLaunchKernelGGL((k_pages_read<TYPE, EL>), grid, dim3(threads_for(pg, rows)), lds, st, pg, b, new_only, log2_up(pg.hd / EL), k, v);
    return hipGetLastError();
}

template <int TYPE>
hipError_t read_both(const PagesView& pg, const BatchView& b, bool new_only, const RowsView& k, const RowsView& v, hipStream_t st) {
    // rows of one width go out in one launch
    const bool wide_k = k.type == FLLM_TYPE_F32, wide_v = v.type == FLLM_TYPE_F32;
    if (!k.p || !v.p || wide_k == wide_v)
        return (k.p ? wide_k : wide_v) ? read<TYPE, 4>(pg, b, new_only, k, v, st) : read<TYPE, 8>(pg, b, new_only, k, v, st);
    const RowsView none{};
    const hipError_t e = wide_k ? read<TYPE, 4>(pg, b, new_only, k, none, st) : read<TYPE, 8>(pg, b, new_only, k, none, st);
    if (e != hipSuccess) return e;
    return wide_v ? read<TYPE, 4>(pg, b, new_only, none, v, st) : read<TYPE, 8>(pg, b, new_only, none, v, st);
}

}  // namespace

hipError_t launch_pages_append(const PagesView& pg, const BatchView& b, const RowsView& k, const RowsView& v, hipStream_t st) {
    if (b.n_rows == 0) return hipSuccess;
    switch (pg.type) {
        case FLLM_TYPE_F16: return append<FLLM_TYPE_F16>(pg, b, k, v, st);
        case FLLM_TYPE_Q8_0: return append<FLLM_TYPE_Q8_0>(pg, b, k, v, st);
        case FLLM_TYPE_Q4_0: return append<FLLM_TYPE_Q4_0>(pg, b, k, v, st);
    }
    return hipErrorNotSupported;
}

hipError_t launch_pages_read(const PagesView& pg, const BatchView& b, bool new_only, const RowsView& k, const RowsView& v,
                             hipStream_t st) {
    if ((new_only ? b.n_new_tiles : b.n_blocks) == 0) return hipSuccess;
    switch (pg.type) {
        case FLLM_TYPE_F16: return read_both<FLLM_TYPE_F16>(pg, b, new_only, k, v, st);
        case FLLM_TYPE_Q8_0: return read_both<FLLM_TYPE_Q8_0>(pg, b, new_only, k, v, st);
        case FLLM_TYPE_Q4_0: return read_both<FLLM_TYPE_Q4_0>(pg, b, new_only, k, v, st);
    }
    return hipErrorNotSupported;
}

}  // namespace fllm
