// draft.hip — drafted tokens checked against the target's probabilities.
#include "pages.hpp"

namespace fllm {

namespace {

// what a weight counts as: positive numbers as themselves, the rest as nothing
__device__ __forceinline__ double counted(double w) { return w > 0.0 ? w : 0.0; }

__global__ __launch_bounds__(1024) void k_draft_verify(DraftView d) {
    __shared__ int s_count, s_token;
    __shared__ double s_sum[1024];
    const int s = blockIdx.x, tid = threadIdx.x;
    const int n = d.counts ? min(max(d.counts[s], 0), d.n_draft) : d.n_draft;
    if (tid == 0) {
        int c = 0;
        for (; c < n; c++) {
            const int t = d.tokens[(int64_t)s * d.n_draft + c];
            if (t < 0 || t >= d.vocab) break;
            const double p = d.target[((int64_t)s * (d.n_draft + 1) + c) * d.target_ld + t];
            const double q = d.draft ? d.draft[((int64_t)s * d.n_draft + c) * d.draft_ld + t] : 1.0;
            if (!((double)d.u_accept[(int64_t)s * d.n_draft + c] * q < p)) break;
        }
        s_count = c;
        s_token = -1;
    }
    __syncthreads();
    const int c = s_count;
    const float* tp = d.target + ((int64_t)s * (d.n_draft + 1) + c) * d.target_ld;
    const float* dp = d.draft && c < n ? d.draft + ((int64_t)s * d.n_draft + c) * d.draft_ld : nullptr;
    const int point = !d.draft && c < n ? d.tokens[(int64_t)s * d.n_draft + c] : -1;
    const int per = (d.vocab + 1023) / 1024, lo = min(d.vocab, tid * per), hi = min(d.vocab, lo + per);
    bool rest = c < n;
    double before = 0.0, total = 0.0;
    for (;;) {
        double sum = 0.0;
        for (int i = lo; i < hi; i++) {
            const double w = !rest ? (double)tp[i] : dp ? (double)tp[i] - (double)dp[i] : (double)tp[i] - (i == point ? 1.0 : 0.0);
            sum += counted(w);
        }
        __syncthreads();
        s_sum[tid] = sum;
        __syncthreads();
        before = total = 0.0;
        for (int i = 0; i < 1024; i++) {
            if (i == tid) before = total;
            total += s_sum[i];
        }
        if (!rest || total > 0.0) break;
        rest = false;
    }
    const double want = (double)d.u_sample[s] * total;
    // the first weight whose running sum passes `want`; were rounding to leave none, the last positive one
    int last = -1, found = -1;
    double run = before;
    for (int i = lo; i < hi && found < 0; i++) {
        const double w = counted(!rest ? (double)tp[i] : dp ? (double)tp[i] - (double)dp[i] : (double)tp[i] - (i == point ? 1.0 : 0.0));
        run += w;
        if (w > 0.0) {
            last = i;
            if (run > want) found = i;
        }
    }
    __shared__ int s_found, s_last;
    if (tid == 0) s_found = d.vocab, s_last = -1;
    __syncthreads();
    if (found >= 0) atomicMin(&s_found, found);
    atomicMax(&s_last, last);
    __syncthreads();
    int* out = d.out_tokens + (int64_t)s * (d.n_draft + 1);
    for (int i = tid; i <= d.n_draft; i += 1024) {
        const int tok = s_found < d.vocab ? s_found : s_last >= 0 ? s_last : d.vocab - 1;
        out[i] = i < c ? d.tokens[(int64_t)s * d.n_draft + i] : i == c ? tok : -1;
    }
    if (tid == 0) d.out_counts[s] = c;
}

}  // namespace

hipError_t launch_draft_verify(const DraftView& d, hipStream_t st) {
    if (d.n_seqs == 0) return hipSuccess;
    hipLaunchKernelGGL(k_draft_verify, dim3(d.n_seqs), dim3(1024), 0, st, d);
    return hipGetLastError();
}

}  // namespace fllm
