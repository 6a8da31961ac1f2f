/*
 * fl_verify.cu — verification of drafted tokens against the target's logits
 * (fl_verify_device).
 *
 * rows: one CTA per logits row takes its maximum (first index) and the sum of
 * exp((l - max) / T).  draw: one CTA per sequence walks the acceptance tests,
 * then draws from the row that stopped it by cumulative sums in 64 bits.
 */
#include <cfloat>
#include <climits>

#include "fl_paged.cuh"

namespace {

constexpr int kThreads = 512;

struct RowStat {
    double z;   /* sum of exp((l - m) / T) */
    float m;    /* largest logit; -infinity: everything masked */
    int32_t best;
};

/* NaN is masked, +infinity is the largest finite value. */
template <typename T>
__device__ __forceinline__ float logit(const T* row, int x)
{
    const float l = fl_to_float(row[x]);
    return l != l ? -INFINITY : fminf(l, FLT_MAX);
}

__device__ __forceinline__ double weight(float l, float m, double inv_t) { return exp(((double)l - (double)m) * inv_t); }

__device__ __forceinline__ double block_sum(double v, double* scratch)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < kThreads / 32; w++) s += scratch[w];
    return s;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(const FlVerify g, RowStat* __restrict__ stat)
{
    __shared__ double s_d[kThreads / 32];
    __shared__ float s_m[kThreads / 32];
    __shared__ int s_i[kThreads / 32];
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s = fl_row_seq(g.row_start, g.n_seqs, row);
    if (s < 0) return;
    const T* l = static_cast<const T*>(g.logits) + row * g.logits_stride;
    float m = -INFINITY;
    int best = 0;
    for (int x = threadIdx.x; x < g.vocab; x += kThreads) {
        const float v = logit(l, x);
        if (v > m) m = v, best = x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
        const int b2 = __shfl_xor_sync(0xffffffffu, best, o);
        if (m2 > m || (m2 == m && b2 < best)) m = m2, best = b2;
    }
    if (lane == 0) s_m[warp] = m, s_i[warp] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; w++)
        if (s_m[w] > m || (s_m[w] == m && s_i[w] < best)) m = s_m[w], best = s_i[w];
    const float t = g.temperature[s];
    double z = 0.0;
    if (t > 0.0f && m > -INFINITY) {
        const double inv_t = 1.0 / (double)t;
        for (int x = threadIdx.x; x < g.vocab; x += kThreads) z += weight(logit(l, x), m, inv_t);
    }
    z = block_sum(z, s_d);
    if (threadIdx.x == 0) stat[row] = RowStat{z, m, best};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_draw_kernel(const FlVerify g, const RowStat* __restrict__ stat)
{
    __shared__ double s_d[kThreads / 32];
    __shared__ double s_run[2];
    __shared__ int s_stop, s_rej, s_tok;
    const int s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r0 = max(g.row_start[s], 0), r1 = min(g.row_start[s + 1], g.n_rows);
    if (r1 <= r0) {
        if (threadIdx.x == 0) g.accepted[s] = 0;
        return;
    }
    const float t = g.temperature[s];
    const bool greedy = !(t > 0.0f);
    const double inv_t = greedy ? 1.0 : 1.0 / (double)t;
    if (warp == 0) {
        int stop = r1 - 1, rej = 0;
        for (int base = r0; base < r1 - 1; base += 32) {
            const int row = base + lane;
            bool ok = true;
            if (row < r1 - 1) {
                const RowStat st = stat[row];
                const int d = g.draft[row];
                ok = d >= 0 && d < g.vocab && st.m > -INFINITY;
                if (ok && greedy) {
                    ok = d == st.best;
                } else if (ok) {
                    float q = 1.0f;
                    if (g.probs) q = g.probs[row * g.probs_stride + d];
                    q = q > 0.0f ? q : 0.0f;
                    const float l = logit(static_cast<const T*>(g.logits) + row * g.logits_stride, d);
                    ok = (double)g.u_accept[row] * (double)q * st.z < weight(l, st.m, inv_t);
                }
            }
            const unsigned bad = __ballot_sync(0xffffffffu, !ok);
            if (bad) {
                stop = base + __ffs(bad) - 1;
                rej = 1;
                break;
            }
        }
        if (lane == 0) s_stop = stop, s_rej = rej, s_tok = -1;
    }
    __syncthreads();
    const int r = s_stop;
    const bool rej = s_rej;
    const RowStat st = stat[r];
    int token = -1;
    if (st.m > -INFINITY) {
        if (greedy) {
            token = st.best;
        } else {
            const T* l = static_cast<const T*>(g.logits) + r * g.logits_stride;
            const float* q = g.probs ? g.probs + r * g.probs_stride : nullptr;
            const int d = g.draft[r];
            bool rest = rej;
            auto w_of = [&](int x) -> double {
                const double e = weight(logit(l, x), st.m, inv_t);
                if (!rest) return e;
                if (!q) return x == d ? 0.0 : e;
                const float qx = q[x] > 0.0f ? q[x] : 0.0f;
                return fmax(e - (double)qx * st.z, 0.0);
            };
            double total = 0.0;
            for (int x = threadIdx.x; x < g.vocab; x += kThreads) total += w_of(x);
            total = block_sum(total, s_d);
            if (rest && !(total > 0.0)) {
                rest = false;
                total = st.z;
            }
            const double goal = (double)g.u_sample[s] * total;
            double run = 0.0;
            int last = -1; /* the last x with weight, should rounding leave the goal above every sum */
            for (int base = 0; base < g.vocab; base += kThreads) {
                const int x = base + threadIdx.x;
                const double w = x < g.vocab ? w_of(x) : 0.0;
                double c = w; /* inclusive scan over the block */
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double u = __shfl_up_sync(0xffffffffu, c, o);
                    if (lane >= o) c += u;
                }
                __syncthreads();
                if (lane == 31) s_d[warp] = c;
                __syncthreads();
                double before = run, all = run;
                for (int i = 0; i < kThreads / 32; i++) {
                    if (i < warp) before += s_d[i];
                    all += s_d[i];
                }
                if (w > 0.0) last = x;
                const bool hit = w > 0.0 && before + c > goal;
                if (threadIdx.x == 0) s_tok = INT_MAX;
                __syncthreads();
                if (hit) atomicMin(&s_tok, x);
                __syncthreads();
                if (s_tok != INT_MAX) break;
                run = all;
            }
            __syncthreads();
            if (s_tok == INT_MAX) {
                __syncthreads();
                if (threadIdx.x == 0) s_tok = -1;
                __syncthreads();
                if (last >= 0) atomicMax(&s_tok, last);
                __syncthreads();
            }
            token = s_tok;
        }
    }
    for (int row = r0 + threadIdx.x; row < r1; row += kThreads)
        g.tokens[row] = row < r ? g.draft[row] : row == r ? token : -1;
    if (threadIdx.x == 0) g.accepted[s] = r - r0;
}

template <typename T>
cudaError_t launch(const FlVerify& v, cudaStream_t st)
{
    RowStat* stat = static_cast<RowStat*>(v.workspace);
    if (v.n_rows > 0) verify_rows_kernel<T><<<v.n_rows, kThreads, 0, st>>>(v, stat);
    verify_draw_kernel<T><<<v.n_seqs, kThreads, 0, st>>>(v, stat);
    return cudaGetLastError();
}

} // namespace

size_t fl_verify_workspace_bytes(int n_rows, int, int) { return (size_t)n_rows * sizeof(RowStat); }

cudaError_t fl_launch_verify(const FlVerify& v, cudaStream_t st)
{
    switch (v.type) {
    case 0: return launch<float>(v, st);
    case 1: return launch<__half>(v, st);
    case 30: return launch<__nv_bfloat16>(v, st);
    default: return cudaErrorInvalidValue;
    }
}
