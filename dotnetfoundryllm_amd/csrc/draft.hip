// draft.hip — drafted tokens checked against the target's probabilities.
//
// Bound: two rows of the vocabulary a sequence (1 MB each way at 128256) and the latency of three dependent
// passes: the kept tokens, the weights' sum, the place of the drawn number in their running sum. One launch:
// every workgroup works the kept tokens out for itself (a few scattered loads), sums some segments of the
// row's weights, and the one of a sequence that finishes last finds the segment and then the id. Sums are in
// 64 bits and in a fixed order. 64 x 152064: 78 MB in 26.5 us (2.9 TB/s; 15 us at a copy's rate, 10 us are the chain
// of dependent loads); one sequence of 128256: 15.8 us, all of it latency.
#include "attn_body.hpp"
#include "pages.hpp"

namespace fllm {

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4a __attribute__((ext_vector_type(4), aligned(4)));  // rows need no alignment beyond their elements'

// what a weight counts as: positive numbers as themselves, the rest as nothing
__device__ __forceinline__ double counted(double w) { return w > 0.0 ? w : 0.0; }

struct Weights {
    const float *t, *d;  // target, draft (null: nothing is taken away)
    int point;           // the id that a certain draft takes 1 away from, -1: none
    bool rest;           // target less draft; else target alone
    __device__ __forceinline__ double of(float p, float q, int i) const {
        if (!rest) return counted((double)p);
        return counted((double)p - (d ? (double)q : i == point ? 1.0 : 0.0));
    }
};

// A thread's ids of a segment: lo + 1024 k + 4 thread + e, 4 k and 4 e; zeros past hi.
struct Ids16 {
    f4a p[4], q[4];
    __device__ __forceinline__ void load(const Weights& w, int lo, int hi) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = lo + 1024 * k + 4 * (int)threadIdx.x;
            p[k] = q[k] = f4a{0.f, 0.f, 0.f, 0.f};
            if (i + 4 <= hi) {
                p[k] = *(const f4a*)(w.t + i);
                if (w.d) q[k] = *(const f4a*)(w.d + i);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (i + e < hi) {
                        p[k][e] = w.t[i + e];
                        if (w.d) q[k][e] = w.d[i + e];
                    }
            }
        }
    }
};

// v + the value that DPP control CTRL moves here in the rows of mask ROWS (elsewhere v + 0)
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double dpp_add(double v) {
    union { double d; int i[2]; } a, b;
    a.d = v;
    b.i[0] = __builtin_amdgcn_update_dpp(0, a.i[0], CTRL, ROWS, 0xF, false);
    b.i[1] = __builtin_amdgcn_update_dpp(0, a.i[1], CTRL, ROWS, 0xF, false);
    return v + b.d;
}

// running sums over the workgroup's 256 threads of N values at once: what lies before this thread's v[k]
// in before[k], each sum in total[k]
template <int N>
__device__ __forceinline__ void scan256(const double v[N], double before[N], double total[N], double (*s_wave)[4]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double run[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        run[k] = dpp_add<0x111>(v[k]);  // row_shr 1, 2, 4, 8: running sums of 16 lanes
        run[k] = dpp_add<0x112>(run[k]);
        run[k] = dpp_add<0x114>(run[k]);
        run[k] = dpp_add<0x118>(run[k]);
        run[k] = dpp_add<DPP_BCAST15, 0xA>(run[k]);
        run[k] = dpp_add<DPP_BCAST31, 0xC>(run[k]);
    }
    __syncthreads();
    if (lane == 63)
        for (int k = 0; k < N; k++) s_wave[k][wave] = run[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; k++) {
        double b = 0.0, all = 0.0;
        for (int w = 0; w < 4; w++) {
            if (w < wave) b += s_wave[k][w];
            all += s_wave[k][w];
        }
        total[k] = all;
        before[k] = b + (run[k] - v[k]);
    }
}

__global__ __launch_bounds__(256) void k_draft_verify(DraftView d, int seg, int n_seg, int runs, double* part, unsigned* cnt) {
    __shared__ double s_wave[4][4], s_want;
    __shared__ int s_seg, s_last, s_found, s_pos, s_id;
    const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int given = d.counts ? d.counts[s] : d.n_draft;
    const float u_sample = d.u_sample[s];

    // the tokens kept, a lane each; every wave finds them by itself
    int c = 0, n = 0;
    for (int i0 = 0; i0 < d.n_draft; i0 += 64) {
        const int i = i0 + lane;
        bool no = true;
        if (i < d.n_draft) {
            const int t = d.tokens[(int64_t)s * d.n_draft + i];
            const float u = d.u_accept[(int64_t)s * d.n_draft + i];
            if (t >= 0 && t < d.vocab) {
                const double p = d.target[((int64_t)s * (d.n_draft + 1) + i) * d.target_ld + t];
                const double q = d.draft ? d.draft[((int64_t)s * d.n_draft + i) * d.draft_ld + t] : 1.0;
                no = !((double)u * q < p);
            }
        }
        n = min(max(given, 0), d.n_draft);
        const unsigned long long b = __ballot(no || i >= n);
        c = b ? min(i0 + __builtin_ctzll(b), n) : min(i0 + 64, n);
        if (b || c == n) break;
    }
    n = min(max(given, 0), d.n_draft);
    Weights w;
    w.t = d.target + ((int64_t)s * (d.n_draft + 1) + c) * d.target_ld;
    w.rest = c < n;
    w.d = d.draft && w.rest ? d.draft + ((int64_t)s * d.n_draft + c) * d.draft_ld : nullptr;
    w.point = !d.draft && w.rest ? d.tokens[(int64_t)s * d.n_draft + c] : -1;

    // these segments' sums: of the weights, and of the target's alone
    const int seg0 = blockIdx.x * runs, seg1 = min(seg0 + runs, n_seg);
    const __amdgpu_buffer_rsrc_t rp = wt_rsrc(part + (int64_t)s * n_seg * 2, (uint32_t)n_seg * 16);
    Ids16 x;
    x.load(w, seg0 * seg, min(seg0 * seg + seg, d.vocab));
    for (int g = seg0; g < seg1; g++) {
        Ids16 next;
        const int lo = g * seg, ahead = (g + 1 < seg1 ? g + 1 : g) * seg;
        next.load(w, ahead, g + 1 < seg1 ? min(ahead + seg, d.vocab) : ahead);
        double sums[2] = {0.0, 0.0}, before2[2];
#pragma unroll
        for (int k = 0; k < 4; k++)
            for (int e = 0; e < 4; e++) {
                sums[0] += w.of(x.p[k][e], x.q[k][e], lo + 1024 * k + 4 * tid + e);
                sums[1] += counted((double)x.p[k][e]);
            }
        scan256<2>(sums, before2, sums, s_wave);
        if (tid == 0) {
            union { double v[2]; u4 u; } both;
            both.v[0] = sums[0];
            both.v[1] = sums[1];
            __builtin_amdgcn_raw_buffer_store_b128(both.u, rp, (uint32_t)g * 16, 0, CPOL_SC1);
        }
        x = next;
    }
    if (tid == 0) {
        wt_complete();
        s_last = __hip_atomic_fetch_add(cnt + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        if (s_last) st_wt_u(cnt + s, 0u);
    }
    __syncthreads();
    if (!s_last) return;

    // the sequence's last workgroup: the segment that the drawn number falls into (a thread each)
    double mine[2] = {0.0, 0.0}, before[2], total[2];
    if (tid < n_seg) {
        const float4 f = ld_wt4(rp, (uint32_t)tid * 16);
        __builtin_memcpy(mine, &f, 16);
    }
    if (tid == 0) s_seg = n_seg, s_pos = -1, s_found = d.vocab, s_id = -1;
    scan256<2>(mine, before, total, s_wave);
    if (w.rest && !(total[0] > 0.0)) {  // nothing left: the target itself
        w.rest = false;
        w.d = nullptr;
    }
    const int kind = w.rest || c == n ? 0 : 1;
    const double own = kind ? mine[1] : mine[0], ahead = kind ? before[1] : before[0];
    const double want = (double)u_sample * (kind ? total[1] : total[0]);
    // the first whose running sum passes `want`; were rounding to leave none, the last positive one
    if (own > 0.0) {
        if (ahead + own > want) atomicMin(&s_seg, tid);
        atomicMax(&s_pos, tid);
    }
    __syncthreads();
    const int at = s_seg < n_seg ? s_seg : s_pos;
    if (tid == at) s_want = want - ahead;
    if (at >= 0) {
        // the id within the segment
        const int a = at * seg, z = min(a + seg, d.vocab);
        x.load(w, a, z);
        double v[4], pre[4], all[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[k] = 0.0;
            for (int e = 0; e < 4; e++) v[k] += w.of(x.p[k][e], x.q[k][e], a + 1024 * k + 4 * tid + e);
        }
        scan256<4>(v, pre, all, s_wave);
        const double past = s_want;
        double base = 0.0;
        int found = d.vocab, last = -1;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            double run = base + pre[k];
            for (int e = 0; e < 4; e++) {
                const int i = a + 1024 * k + 4 * tid + e;
                const double y = w.of(x.p[k][e], x.q[k][e], i);
                run += y;
                if (y > 0.0) {
                    last = i;
                    if (run > past && found == d.vocab) found = i;
                }
            }
            base += all[k];
        }
        if (found < d.vocab) atomicMin(&s_found, found);
        if (last >= 0) atomicMax(&s_id, last);
        __syncthreads();
    }
    const int token = s_found < d.vocab ? s_found : s_id >= 0 ? s_id : d.vocab - 1;
    int* out = d.out_tokens + (int64_t)s * (d.n_draft + 1);
    for (int i = tid; i <= d.n_draft; i += 256) out[i] = i < c ? d.tokens[(int64_t)s * d.n_draft + i] : i == c ? token : -1;
    if (tid == 0) d.out_counts[s] = c;
}

}  // namespace

// Segments of a row: of 1024 ids (4 a thread) at least and 4096 (16 a thread) at most, shorter ones while they leave
// every CU no more than a few workgroups over all sequences; up to 256 of them (a thread each in the last workgroup).
// A workgroup takes `runs` of them in a row, the next one's loads under way while one is summed, so that two
// workgroups a CU remain: each begins with the same three dependent loads. 64 x 152064: 1 run 37.5 us, 2: 29.7,
// 3: 27.4, 4: 26.9, 6: 26.4, 10: 29.8; 1 x 128256 (126 segments): 1 run 16.5 us, 2: 16.9, 4: 19.8.
int draft_segments(int n_seqs, int vocab, int n_cu, int* seg, int* runs) {
    int k = (int)((int64_t)n_seqs * vocab / ((int64_t)4 * n_cu * 1024)) + 1;
    k = k > 4 ? 4 : k;
    while (k < 4 && (vocab + 1024 * k - 1) / (1024 * k) > 256) k++;
    *seg = 1024 * k;
    const int n_seg = (vocab + *seg - 1) / *seg;
    const int64_t r = (int64_t)n_seqs * n_seg / (2 * n_cu);
    *runs = r < 1 ? 1 : r < n_seg ? (int)r : n_seg;
    return n_seg;
}

hipError_t launch_draft_verify(const DraftView& d, int seg, int n_seg, int runs, double* part, unsigned* cnt, hipStream_t st) {
    for (int s0 = 0; s0 < d.n_seqs; s0 += 65535) {  // the grid's second dimension ends at 65535
        DraftView v = d;
        v.n_seqs = d.n_seqs - s0 < 65535 ? d.n_seqs - s0 : 65535;
        const int64_t n1 = d.n_draft + 1;
        v.target += s0 * n1 * d.target_ld;
        if (v.draft) v.draft += (int64_t)s0 * d.n_draft * d.draft_ld;
        if (v.tokens) v.tokens += (int64_t)s0 * d.n_draft;
        if (v.counts) v.counts += s0;
        if (v.u_accept) v.u_accept += (int64_t)s0 * d.n_draft;
        v.u_sample += s0;
        v.out_tokens += s0 * n1;
        v.out_counts += s0;
        hipLaunchKernelGGL(k_draft_verify, dim3((n_seg + runs - 1) / runs, v.n_seqs), dim3(256), 0, st, v, seg, n_seg, runs, part + (int64_t)s0 * n_seg * 2, cnt + s0);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace fllm
