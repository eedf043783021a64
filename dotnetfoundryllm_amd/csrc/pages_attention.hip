// pages_attention.hip — attention of new tokens over the pages of their sequences.
#include "pages.hpp"

namespace fllm {

namespace {

template <int TYPE>
__device__ __forceinline__ float cell_value(const PagesView& pg, const uint8_t* cell, int kind, int d, int pos) {
    const int P = 1 << pg.page_log2, blk = d >> 5, e = d & 31;
    if (TYPE == FLLM_TYPE_F16) return half_exact(((const uint16_t*)cell)[kind ? d * P + pos : (blk * P + pos) * 32 + e]);
    const float s = half_exact(*(const uint16_t*)(cell + pg.scale_off + 2 * (blk * P + pos)));
    if (TYPE == FLLM_TYPE_Q8_0) return (float)(int8_t)cell[kind ? d * P + pos : (blk * P + pos) * 32 + e] * s;
    const int c = cell[kind ? (blk * 16 + (e & 15)) * P + pos : (blk * P + pos) * 16 + (e & 15)];
    return (float)((e < 16 ? c & 15 : c >> 4) - 8) * s;
}

// One workgroup per new token and query head; a wave per key, lane l holding the elements l + 64 i.
template <int TYPE>
__global__ __launch_bounds__(256) void k_pages_attention(PagesView pg, BatchView b, RowsView q, RowsView out, float scale,
                                                         float softcap) {
    __shared__ float s_o[4][256], s_m[4], s_l[4];
    const int row = blockIdx.x, h = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int lo = 0, hi = b.n_seqs - 1;
    while (lo < hi) {  // the last sequence that starts at or before this row and has one
        const int mid = (lo + hi + 1) >> 1;
        if (b.seqs[mid].x <= row) lo = mid;
        else hi = mid - 1;
    }
    const int4 sq = b.seqs[lo];
    const int pos = sq.z - sq.y + (row - sq.x), kvh = h / (b.n_heads / pg.nkv);
    const int64_t first = (int64_t)pos - b.window + 1;
    const int* table = b.tables + (int64_t)lo * b.tab_w;
    float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    for (int i = 0; i < 4; i++) qv[i] = lane + 64 * i < pg.hd ? row_elem(q, row * q.ld + h * pg.hd + lane + 64 * i) : 0.f;
    for (int j = (int)(first > 0 ? first : 0) + wave; j <= pos; j += 4) {
        const uint64_t cell = ((uint64_t)table[j >> pg.page_log2] * pg.nkv + kvh) * pg.cell;
        const int p = j & ((1 << pg.page_log2) - 1);
        float s = 0.f;
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < pg.hd) s = fmaf(qv[i], cell_value<TYPE>(pg, pg.k + cell, 0, lane + 64 * i, p), s);
        for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x);
        s *= scale;
        if (softcap > 0.f) s = softcap * tanhf(s / softcap);
        const float nm = fmaxf(m, s), a = expf(m - nm), w = expf(s - nm);
        m = nm;
        l = l * a + w;
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < pg.hd) o[i] = o[i] * a + w * cell_value<TYPE>(pg, pg.v + cell, 1, lane + 64 * i, p);
    }
    for (int i = 0; i < 4; i++) s_o[wave][lane + 64 * i] = o[i];
    if (lane == 0) s_m[wave] = m, s_l[wave] = l;
    __syncthreads();
    const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float sum = 0.f, acc = 0.f;
    for (int w = 0; w < 4; w++) {
        const float f = s_l[w] > 0.f ? expf(s_m[w] - top) : 0.f;
        sum += f * s_l[w];
        if (threadIdx.x < pg.hd) acc += f * s_o[w][threadIdx.x];
    }
    if (threadIdx.x < pg.hd) row_store(out, row * out.ld + h * pg.hd + threadIdx.x, acc / sum);
}

}  // namespace

hipError_t launch_pages_attention(const PagesView& pg, const BatchView& b, const RowsView& q, const RowsView& out,
                                  float scale, float softcap, hipStream_t st) {
    if (b.n_rows == 0) return hipSuccess;
    const dim3 grid(b.n_rows, b.n_heads);
    switch (pg.type) {
        case FLLM_TYPE_F16: hipLaunchKernelGGL(k_pages_attention<FLLM_TYPE_F16>, grid, dim3(256), 0, st, pg, b, q, out, scale, softcap); break;
        case FLLM_TYPE_Q8_0: hipLaunchKernelGGL(k_pages_attention<FLLM_TYPE_Q8_0>, grid, dim3(256), 0, st, pg, b, q, out, scale, softcap); break;
        case FLLM_TYPE_Q4_0: hipLaunchKernelGGL(k_pages_attention<FLLM_TYPE_Q4_0>, grid, dim3(256), 0, st, pg, b, q, out, scale, softcap); break;
        default: return hipErrorNotSupported;
    }
    return hipGetLastError();
}

}  // namespace fllm
