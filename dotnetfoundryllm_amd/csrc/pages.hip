// pages.hip — rows into and out of the pages of the paged K/V cache.
//
// A workgroup takes the positions of one page that the call covers, for one kv head and one of K and
// V: up to page_size rows of head_dim. Both kernels are bound by memory traffic for many rows and by the
// launch for few. K keeps the rows' direction, so its codes go straight to their place, 8 lanes to a
// block of 32. V is stored with the positions along the row (what the attention's second product
// reads), so its codes are turned in LDS and leave as runs of positions, 16 bytes at a time where the
// run covers them.
#include "pages.hpp"

namespace fllm {

namespace {

struct Tile {
    int off, n;       // first position in the page, number of positions
    int64_t row;      // their first row in the dense matrix
    uint64_t cell;    // the cell's offset
};

// The tile of sequence s that workgroup column bx covers; false where it covers none.
__device__ __forceinline__ bool tile_of(const PagesView& pg, const BatchView& b, bool new_only, int s, int bx, int head,
                                        Tile* t) {
    const int4 q = b.seqs[s];
    const int first = new_only ? q.z - q.y : 0;
    const int pb = (first >> pg.page_log2) + bx;
    const int lo = max(first, pb << pg.page_log2), hi = min(q.z, (pb + 1) << pg.page_log2);
    if (lo >= hi) return false;
    t->off = lo - (pb << pg.page_log2);
    t->n = hi - lo;
    t->row = (int64_t)(new_only ? q.x : q.w) + (lo - first);
    t->cell = ((uint64_t)b.tables[(int64_t)s * b.tab_w + pb] * pg.nkv + head) * pg.cell;
    return true;
}

__device__ __forceinline__ void load4(const RowsView& r, int64_t i, float x[4]) {
    if (r.type == FLLM_TYPE_F32) {
        const float4 f = *(const float4*)(r.p + 4 * i);
        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
        return;
    }
    const uint2 u = *(const uint2*)(r.p + 2 * i);
    const uint32_t h[4] = {u.x & 0xFFFFu, u.x >> 16, u.y & 0xFFFFu, u.y >> 16};
    for (int e = 0; e < 4; e++) x[e] = r.type == FLLM_TYPE_F16 ? half_exact(h[e]) : bf16_exact(h[e]);
}

__device__ __forceinline__ uint32_t half_bits(float f) {
    const _Float16 h = (_Float16)f;
    uint16_t u;
    __builtin_memcpy(&u, &h, 2);
    return u;
}

__device__ __forceinline__ void store4(const RowsView& r, int64_t i, const float x[4]) {
    if (r.type == FLLM_TYPE_F32) {
        *(float4*)(r.p + 4 * i) = make_float4(x[0], x[1], x[2], x[3]);
        return;
    }
    uint32_t h[4];
    for (int e = 0; e < 4; e++) h[e] = r.type == FLLM_TYPE_F16 ? half_bits(x[e]) : bf16_round(x[e]);
    *(uint2*)(r.p + 2 * i) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

// The integer nearest to x / d (ties to even), clamped: the rounded product with the reciprocal is at
// most one off, and the remainder x - c d (exact in one fma: c d has 19 bits) says in which
// direction. A float32 division would round a quotient next to a tie onto it.
__device__ __forceinline__ int code_of(float x, float d, float inv, float half, int lo, int hi) {
    const float c = fminf(fmaxf(rintf(x * inv), -300.0f), 300.0f);
    const float r = fmaf(-c, d, x);
    const float s = d < 0.0f ? -r : r;  // remainder in units of |d|
    float q = c;
    if (s > half || (s == half && ((int)c & 1))) q += 1.0f;
    else if (s < -half || (s == -half && ((int)c & 1))) q -= 1.0f;
    return (int)fminf(fmaxf(q, (float)lo), (float)hi);
}

// The scale of a block of 32 over its 8 lanes, 4 elements each: its bits in half precision.
template <int TYPE>
__device__ __forceinline__ uint32_t block_scale(const float x[4], int e) {
    // order by magnitude, then by the lower index; the sign rides in the low bit. A NaN or an infinity
    // has the largest magnitude bits, so it leads.
    unsigned long long key = 0;
    for (int i = 0; i < 4; i++) {
        const uint32_t u = __float_as_uint(x[i]);
        const unsigned long long k = (unsigned long long)(u & 0x7FFFFFFFu) << 32 | (unsigned)(31 - (4 * e + i)) << 1 | u >> 31;
        key = k > key ? k : key;
    }
    for (int o = 1; o < 8; o <<= 1) {
        const unsigned long long k = __shfl_xor(key, o);
        key = k > key ? k : key;
    }
    const float m = __uint_as_float((uint32_t)(key >> 32));
    if (!(m < __uint_as_float(0x7F800000u))) return 0x7E00u;  // not finite: a NaN scale
    const float d = TYPE == FLLM_TYPE_Q8_0 ? m / 127.0f : m * ((key & 1) ? 0.125f : -0.125f);
    const uint32_t h = half_bits(d);
    return (h & 0x7FFFu) == 0x7C00u ? (h & 0x8000u) | 0x7BFFu : h;
}

template <int TYPE>
__global__ __launch_bounds__(256) void k_pages_append(PagesView pg, BatchView b, RowsView rk, RowsView rv) {
    extern __shared__ __align__(16) uint8_t turned[];
    const int head = blockIdx.z >> 1, kind = blockIdx.z & 1;
    const int P = 1 << pg.page_log2, nb = pg.hd >> 5;
    const RowsView& src = kind ? rv : rk;
    constexpr int ESZ = TYPE == FLLM_TYPE_F16 ? 2 : 1;
    const int pitch = P * ESZ + 16;  // of a V row in LDS
    for (int s = blockIdx.y; s < b.n_seqs; s += gridDim.y) {
        Tile t;
        if (!tile_of(pg, b, true, s, blockIdx.x, head, &t)) continue;
        uint8_t* cell = (kind ? pg.v : pg.k) + t.cell;
        const int e = threadIdx.x & 7;
        for (int u = threadIdx.x >> 3; u < t.n * nb; u += blockDim.x >> 3) {
            const int i = u % t.n, blk = u / t.n, pos = t.off + i;
            float x[4];
            load4(src, (t.row + i) * src.ld + head * pg.hd + blk * 32 + 4 * e, x);
            uint32_t c[4];
            if (TYPE == FLLM_TYPE_F16) {
                for (int j = 0; j < 4; j++) c[j] = half_bits(x[j]);
            } else {
                const uint32_t h = block_scale<TYPE>(x, e);
                const float d = half_exact(h);
                const bool live = d != 0.0f && d == d;
                const float inv = live ? 1.0f / d : 0.0f, half = 0.5f * fabsf(d);
                for (int j = 0; j < 4; j++) {
                    const int q = !live ? 0 : TYPE == FLLM_TYPE_Q8_0 ? code_of(x[j], d, inv, half, -127, 127)
                                                                     : code_of(x[j], d, inv, half, -8, 7);
                    c[j] = TYPE == FLLM_TYPE_Q8_0 ? (uint32_t)q & 0xFFu : (uint32_t)(q + 8);
                }
                if (e == 0) *(uint16_t*)(cell + pg.scale_off + 2 * (blk * P + pos)) = (uint16_t)h;
            }
            if (TYPE == FLLM_TYPE_Q4_0) {  // the upper 16 elements' codes join the lower ones' bytes
                for (int j = 0; j < 4; j++) c[j] |= (uint32_t)__shfl_down(c[j], 4, 8) << 4;
                if (e >= 4) continue;
            }
            if (kind == 0) {
                if (TYPE == FLLM_TYPE_F16)
                    *(uint2*)(cell + 2 * ((blk * P + pos) * 32 + 4 * e)) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
                else
                    *(uint32_t*)(cell + (blk * P + pos) * (TYPE == FLLM_TYPE_Q4_0 ? 16 : 32) + 4 * e) =
                        c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
            } else {
                for (int j = 0; j < 4; j++) {
                    uint8_t* at = turned + (blk * (TYPE == FLLM_TYPE_Q4_0 ? 16 : 32) + 4 * e + j) * pitch + pos * ESZ;
                    if (TYPE == FLLM_TYPE_F16) *(uint16_t*)at = (uint16_t)c[j];
                    else *at = (uint8_t)c[j];
                }
            }
        }
        if (kind == 0) continue;
        __syncthreads();
        const int rows = TYPE == FLLM_TYPE_Q4_0 ? pg.hd / 2 : pg.hd, chunks = P * ESZ / 16, per = 16 / ESZ;
        for (int u = threadIdx.x; u < rows * chunks; u += blockDim.x) {
            const int row = u / chunks, c = u % chunks, lo = max(t.off, c * per), hi = min(t.off + t.n, (c + 1) * per);
            if (lo >= hi) continue;
            const uint8_t* from = turned + row * pitch;
            uint8_t* to = cell + row * P * ESZ;
            if (hi - lo == per) {
                *(uint4*)(to + c * 16) = *(const uint4*)(from + c * 16);
            } else {
                for (int i = lo; i < hi; i++) {
                    if (TYPE == FLLM_TYPE_F16) ((uint16_t*)to)[i] = ((const uint16_t*)from)[i];
                    else to[i] = from[i];
                }
            }
        }
        __syncthreads();
    }
}

template <int TYPE>
__global__ __launch_bounds__(256) void k_pages_read(PagesView pg, BatchView b, bool new_only, RowsView rk, RowsView rv) {
    extern __shared__ __align__(16) uint8_t turned[];
    const int head = blockIdx.z >> 1, kind = blockIdx.z & 1;
    const RowsView& dst = kind ? rv : rk;
    if (!dst.p) return;
    const int P = 1 << pg.page_log2, nb = pg.hd >> 5;
    constexpr int ESZ = TYPE == FLLM_TYPE_F16 ? 2 : 1;
    const int pitch = P * ESZ + 16;
    for (int s = blockIdx.y; s < b.n_seqs; s += gridDim.y) {
        Tile t;
        if (!tile_of(pg, b, new_only, s, blockIdx.x, head, &t)) continue;
        const uint8_t* cell = (kind ? pg.v : pg.k) + t.cell;
        if (kind) {
            const int rows = TYPE == FLLM_TYPE_Q4_0 ? pg.hd / 2 : pg.hd, chunks = P * ESZ / 16;
            for (int u = threadIdx.x; u < rows * chunks; u += blockDim.x)
                *(uint4*)(turned + (u / chunks) * pitch + (u % chunks) * 16) = *(const uint4*)(cell + 16 * u);
            __syncthreads();
        }
        const int e = threadIdx.x & 7;
        for (int u = threadIdx.x >> 3; u < t.n * nb; u += blockDim.x >> 3) {
            const int i = u / nb, blk = u % nb, pos = t.off + i;
            float x[4];
            if (TYPE == FLLM_TYPE_F16) {
                for (int j = 0; j < 4; j++)
                    x[j] = half_exact(kind ? *(const uint16_t*)(turned + (blk * 32 + 4 * e + j) * pitch + 2 * pos)
                                           : ((const uint16_t*)cell)[(blk * P + pos) * 32 + 4 * e + j]);
            } else {
                const float d = half_exact(*(const uint16_t*)(cell + pg.scale_off + 2 * (blk * P + pos)));
                const int per = TYPE == FLLM_TYPE_Q4_0 ? 16 : 32, e4 = 4 * e & (per - 1);
                uint32_t w = 0;
                if (kind == 0) w = *(const uint32_t*)(cell + (blk * P + pos) * per + e4);
                else
                    for (int j = 0; j < 4; j++) w |= (uint32_t)turned[(blk * per + e4 + j) * pitch + pos] << 8 * j;
                for (int j = 0; j < 4; j++) {
                    const uint32_t c = w >> 8 * j & 0xFFu;
                    const int q = TYPE == FLLM_TYPE_Q8_0 ? (int)(int8_t)c : (int)(e < 4 ? c & 15u : c >> 4) - 8;
                    x[j] = (float)q * d;
                }
            }
            store4(dst, (t.row + i) * dst.ld + head * pg.hd + blk * 32 + 4 * e, x);
        }
        __syncthreads();
    }
}

// A tile of few rows has little work for 256 threads: one wave starts sooner and leaves the CU to others.
int threads_for(const PagesView& pg, int rows) { return rows * (pg.hd >> 5) * 8 <= 64 ? 64 : 256; }

size_t turned_bytes(const PagesView& pg) {
    const size_t rows = pg.type == FLLM_TYPE_Q4_0 ? pg.hd / 2 : pg.hd, esz = pg.type == FLLM_TYPE_F16 ? 2 : 1;
    return rows * (((size_t)1 << pg.page_log2) * esz + 16);
}

template <typename K>
hipError_t lds_limit(K kernel, size_t bytes) {
    return bytes <= 65536 ? hipSuccess
                          : hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

}  // namespace

hipError_t launch_pages_append(const PagesView& pg, const BatchView& b, const RowsView& k, const RowsView& v, hipStream_t st) {
    if (b.n_rows == 0) return hipSuccess;
    const dim3 grid(b.new_blocks, b.n_seqs < 65535 ? b.n_seqs : 65535, 2 * pg.nkv);
    const int thr = threads_for(pg, b.n_rows <= b.n_seqs ? 1 : 1 << pg.page_log2);
    const size_t lds = turned_bytes(pg);
#define FLLM_APPEND(T)                                                                       \
    case T: {                                                                                \
        hipError_t e = lds_limit(k_pages_append<T>, lds);                                    \
        if (e != hipSuccess) return e;                                                       \
        hipLaunchKernelGGL(k_pages_append<T>, grid, dim3(thr), lds, st, pg, b, k, v);        \
        return hipGetLastError();                                                            \
    }
    switch (pg.type) {
        FLLM_APPEND(FLLM_TYPE_F16)
        FLLM_APPEND(FLLM_TYPE_Q8_0)
        FLLM_APPEND(FLLM_TYPE_Q4_0)
    }
#undef FLLM_APPEND
    return hipErrorNotSupported;
}

hipError_t launch_pages_read(const PagesView& pg, const BatchView& b, bool new_only, const RowsView& k, const RowsView& v,
                             hipStream_t st) {
    const int blocks = new_only ? b.new_blocks : b.all_blocks;
    if (blocks == 0) return hipSuccess;
    const dim3 grid(blocks, b.n_seqs < 65535 ? b.n_seqs : 65535, 2 * pg.nkv);
    const int thr = threads_for(pg, new_only && b.n_rows <= b.n_seqs ? 1 : 1 << pg.page_log2);
    const size_t lds = turned_bytes(pg);
#define FLLM_READ(T)                                                                              \
    case T: {                                                                                     \
        hipError_t e = lds_limit(k_pages_read<T>, lds);                                           \
        if (e != hipSuccess) return e;                                                            \
        hipLaunchKernelGGL(k_pages_read<T>, grid, dim3(thr), lds, st, pg, b, new_only, k, v);     \
        return hipGetLastError();                                                                 \
    }
    switch (pg.type) {
        FLLM_READ(FLLM_TYPE_F16)
        FLLM_READ(FLLM_TYPE_Q8_0)
        FLLM_READ(FLLM_TYPE_Q4_0)
    }
#undef FLLM_READ
    return hipErrorNotSupported;
}

}  // namespace fllm
