/*
 * fl_verify.cu — verification of drafted tokens against the target's logits
 * (fl_verify_device).
 *
 * Bound by reading the logits once; two kernels, the second started early and
 * waiting for the first (programmatic dependent launch):
 *  rows:   per (row, chunk of 4096 entries) the maximum and the sum of exp((l -
 *          max) / T), exponentials in fp32; the first index of the maximum where
 *          the sequence is greedy;
 *  finish: a cluster of 8 CTAs per sequence, each of whose 64 warps has a
 *          contiguous range of the vocabulary.  Every CTA repeats the acceptance
 *          tests (a few rows of a few partials); then over the row that the
 *          sequence stopped at: the sum of the exponentials, the sum of
 *          max(p - q, 0), which needs the first one's total, and the entry that
 *          the draw falls into, looked for by the warp whose range holds it.
 *          Sums go around by distributed shared memory.
 * The draw compares with cumulative sums of up to 2^24 entries, whose borders
 * lie closer than fp32 resolves: the second kernel's exponentials and sums are
 * in 64 bits.  The acceptance tests compare single probabilities, for which the
 * fp32 exponentials' 2^-22 is enough.
 */
#include <cooperative_groups.h>

#include <cfloat>
#include <climits>

#include "fl_paged.cuh"

namespace {

constexpr int kThreads = 128, kChunk = 4096;
constexpr int kCluster = 8, kFinThreads = 256, kFinWarps = kFinThreads / 32;

struct RowPart { /* of a row's chunk */
    float m, z;
    int32_t best, pad;
};
struct Decision { /* of a sequence */
    double z;    /* sum of exp((l - m) / T) over the row, exponentials in fp32 */
    float m;
    int32_t row; /* that it stopped at */
    int32_t rej, best;
};

__host__ __device__ __forceinline__ int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

/* An infinite temperature is the largest finite one, at which logits of the usual size weigh the same too: divided by
 * infinity, masked ones would be NaN. */
__device__ __forceinline__ float temperature_of(const FlVerify& g, int s)
{
    const float t = g.temperature[s];
    return t > FLT_MAX ? FLT_MAX : t; /* NaN stays: greedy */
}

/* NaN is masked, +infinity is the largest finite value. */
__device__ __forceinline__ float clean(float l) { return l != l ? -INFINITY : fminf(l, FLT_MAX); }

/* Exponentials in 64 bits as 2^(k / 256): k = n + f, |f| <= 1/2; 2^(n / 256) from
 * a table of 256 and an exponent, 2^(f / 256) by its Taylor series to f^3 (the
 * next term is below 2^-42 of the value; a draw's borders are some 2^-20 apart).
 * 64-bit operations are slow, so they are few (the finishing kernel keeps their pipe
 * busy 21 % of the cycles, 45 % on the busiest SM): with b whole, one FMA
 * against 1.5 2^52 + b rounds k = l A + b, one sum takes n away, one FMA gives f.
 * A table of 32 with a copy per lane, free of bank conflicts but with a longer
 * series, took 78 us for a call of 64 sequences where this takes 66. */
constexpr int kTabBits = 8, kTab = 1 << kTabBits;
constexpr double kL = 0.69314718055994531 / kTab, kUnit = kTab * 1.4426950408889634;
struct Table {
    double v[kTab];
};
constexpr Table make_table()
{
    Table t{};
    for (int i = 0; i < kTab; i++) {
        double p = 1.0; /* e^(i kL), i kL < 0.7 */
        for (int k = 20; k > 0; k--) p = 1.0 + p * (kL * i) / k;
        t.v[i] = p;
    }
    return t;
}
__device__ const Table c_table = make_table();

__device__ __forceinline__ double series(double f)
{
    return fma(fma(fma(kL * kL * kL / 6.0, f, kL * kL / 2.0), f, kL), f, 1.0);
}

struct Exp64 {
    double a, bm;        /* A = 256 log2(e) / T; magic + b */
    const double* table; /* in shared memory */
    float least;         /* logits below count as masked */
    /* the value is p * scale: a caller that sums uses one FMA */
    __device__ __forceinline__ void operator()(float l, double& p, double& scale) const
    {
        const double x = (double)(l < least ? -INFINITY : l), t = fma(x, a, bm);
        const double f = fma(x, a, bm - t);
        const int n = __double2loint(t); /* k rounded, while it fits; l = -infinity gives t = -infinity */
        p = series(f);
        const double e = table[n & (kTab - 1)];
        scale = __hiloint2double(__double2hiint(e) + ((n >> kTabBits) << 20), __double2loint(e));
        if (!(t > 6755399441055744.0 - kTab * 1021.0)) p = scale = 0.0; /* below 2^-1021; masked */
    }
    __device__ __forceinline__ double value(float l) const
    {
        double p, scale;
        (*this)(l, p, scale);
        return p * scale;
    }
};
__device__ __forceinline__ void exp64_table(double* table)
{
    for (int i = threadIdx.x; i < kTab; i += blockDim.x) table[i] = c_table.v[i];
}
/* e^((l - m) / T) up to a factor 2^(c / 256), |c| <= 1/2, common to all l.  From
 * |m| A = 2^40 on, neighbouring floats differ by 2^16 in k: only the maximum's
 * equals have weight. */
__device__ __forceinline__ Exp64 exp64_of(float m, float t, const double* table)
{
    const double a = kUnit / (double)t, b = (double)m * a;
    if (fabs(b) < 1099511627776.0) return Exp64{a, 6755399441055744.0 - rint(b), table, -INFINITY};
    return Exp64{fabs(1.0 / (double)m), 6755399441055744.0 - (m > 0.0f ? 1.0 : -1.0), table, m};
}
/* e^(x / T) for x <= 0, itself */
__device__ __forceinline__ double exp_over(double x, float t, const double* table)
{
    const double k = fmax(x * (kUnit / (double)t), -(double)kTab * 1100.0), n = rint(k);
    const int i = (int)n;
    return i <= -kTab * 1021 ? 0.0 : series(k - n) * table[i & (kTab - 1)] * __hiloint2double((1023 + (i >> kTabBits)) << 20, 0);
}

__device__ __forceinline__ double warp_sum(double v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

/* The larger of each half's two numbers, NaN losing. */
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __half)
{
    const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __nv_bfloat16)
{
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ float2 halves(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
__device__ __forceinline__ float2 halves(uint32_t w, __nv_bfloat16)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

/* The largest of 16 bytes of logits, NaN losing; -infinity if there is no other. */
template <typename T>
__device__ __forceinline__ float max_of(const uint4& u)
{
    if constexpr (sizeof(T) == 4) {
        return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
                     fmaxf(__uint_as_float(u.z), fmaxf(__uint_as_float(u.w), -INFINITY)));
    } else {
        const float2 f = halves(max2(max2(u.x, u.y, T()), max2(u.z, u.w, T()), T()), T());
        return fmaxf(fmaxf(f.x, f.y), -INFINITY);
    }
}

/* Sum of 2^((l - m) c) over 16 bytes of logits; NaN if one is NaN or infinite. */
template <typename T>
__device__ __forceinline__ float sum_of(const uint4& u, float m, float c)
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float z = 0.0f, z1 = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            z += fl_ex2((__uint_as_float(w[i]) - m) * c);
        } else {
            const float2 f = halves(w[i], T());
            z += fl_ex2((f.x - m) * c);
            z1 += fl_ex2((f.y - m) * c);
        }
    }
    return z + z1;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(const FlVerify g)
{
    constexpr int VE = 16 / sizeof(T), NV = kChunk / (VE * kThreads);
    __shared__ float s_m[kThreads / 32], s_z[kThreads / 32];
    __shared__ int s_i[kThreads / 32];
    const int chunk = blockIdx.y, row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    fl_pdl_trigger();
    const T* l = static_cast<const T*>(g.logits) + row * g.logits_stride;
    const int x0 = chunk * kChunk, x1 = min(g.vocab, x0 + kChunk), n = x1 - x0;
    /* the thread's entries, all loaded before any is used: an unaligned start, then 16 bytes at a time, then the end */
    const int head = min(n, (int)((16 - reinterpret_cast<uintptr_t>(l + x0) % 16) % 16 / sizeof(T)));
    const int nv = (n - head) / VE, tail = head + nv * VE + threadIdx.x;
    const uint4* v = reinterpret_cast<const uint4*>(l + x0 + head);
    uint4 u[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int at = threadIdx.x + i * kThreads;
        if (at < nv) u[i] = __ldg(v + at);
    }
    float ends[2] = {-INFINITY, -INFINITY};
    if ((int)threadIdx.x < head) ends[0] = clean(fl_to_float(l[x0 + threadIdx.x]));
    if (tail < n) ends[1] = clean(fl_to_float(l[x0 + tail]));
    const int s = fl_row_seq(g.row_start, g.n_seqs, row); /* while they are under way */
    if (s < 0) return;
    const float t = temperature_of(g, s);
    float m = fmaxf(ends[0], ends[1]);
#pragma unroll
    for (int i = 0; i < NV; i++)
        if ((int)threadIdx.x + i * kThreads < nv) m = fmaxf(m, max_of<T>(u[i]));
    m = fminf(m, FLT_MAX);
    const float mine = m;
    m = fl_warp_max(m);
    /* its first index, looked for by the threads that hold it */
    int best = INT_MAX;
    if (!(t > 0.0f) && mine == m && m > -INFINITY) {
        if (ends[1] == m) best = x0 + tail;
#pragma unroll
        for (int i = NV - 1; i >= 0; i--) {
            if ((int)threadIdx.x + i * kThreads >= nv) continue;
            const T* e = reinterpret_cast<const T*>(&u[i]);
#pragma unroll
            for (int j = VE - 1; j >= 0; j--)
                if (clean(fl_to_float(e[j])) == m) best = x0 + head + (threadIdx.x + i * kThreads) * VE + j;
        }
        if (ends[0] == m) best = x0 + threadIdx.x;
    }
    best = __reduce_min_sync(0xffffffffu, best);
    /* the thread's sum against its own maximum, brought to the warp's, then to the chunk's */
    float z = 0.0f;
    if (t > 0.0f && mine > -INFINITY) {
        const float c = fminf(1.44269504f / t, FLT_MAX);
#pragma unroll
        for (int i = 0; i < NV; i++)
            if ((int)threadIdx.x + i * kThreads < nv) z += sum_of<T>(u[i], mine, c);
        if (z != z || mine == FLT_MAX) { /* a NaN or an infinity among them: one by one */
            z = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if ((int)threadIdx.x + i * kThreads >= nv) continue;
                const T* e = reinterpret_cast<const T*>(&u[i]);
#pragma unroll
                for (int j = 0; j < VE; j++) z += fl_ex2((clean(fl_to_float(e[j])) - mine) * c);
            }
        }
        z += fl_ex2((ends[0] - mine) * c) + fl_ex2((ends[1] - mine) * c);
        z *= fl_ex2((mine - m) * c);
    }
    z = fl_warp_sum(z);
    if (lane == 0) s_m[warp] = m, s_z[warp] = z, s_i[warp] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        float M = -INFINITY, Z = 0.0f;
        int B = INT_MAX;
        for (int w = 0; w < kThreads / 32; w++)
            if (s_m[w] > M || (s_m[w] == M && s_i[w] < B)) M = s_m[w], B = s_i[w];
        for (int w = 0; w < kThreads / 32; w++)
            if (s_m[w] > -INFINITY && t > 0.0f) Z += s_z[w] * fl_ex2((s_m[w] - M) * fminf(1.44269504f / t, FLT_MAX));
        static_cast<RowPart*>(g.workspace)[(size_t)row * gridDim.y + chunk] = RowPart{M, Z, B, 0};
    }
}

/* A row's maximum, first index of it and sum, by a warp from its chunks: up to
 * 128 of them are loaded at once, more a second time.  Not __restrict__: the first
 * kernel writes them while this one is already running, so they are not constant
 * for its length, as loads that this allows would take for granted. */
__device__ __forceinline__ Decision merge_row(const RowPart* part, int chunks, float t, const double* table)
{
    const int lane = threadIdx.x & 31;
    Decision d{0.0, -INFINITY, 0, 0, INT_MAX};
    RowPart p[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int c = lane + 32 * i;
        p[i] = c < chunks ? part[c] : RowPart{-INFINITY, 0.0f, INT_MAX, 0};
    }
    auto take = [&](const RowPart& r) {
        if (r.m > d.m || (r.m == d.m && r.best < d.best)) d.m = r.m, d.best = r.best;
    };
#pragma unroll
    for (int i = 0; i < 4; i++) take(p[i]);
    for (int c = lane + 128; c < chunks; c += 32) take(part[c]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, d.m, o);
        const int b2 = __shfl_xor_sync(0xffffffffu, d.best, o);
        if (m2 > d.m || (m2 == d.m && b2 < d.best)) d.m = m2, d.best = b2;
    }
    if (t > 0.0f && d.m > -INFINITY) {
        auto add = [&](const RowPart& r) {
            if (r.m > -INFINITY) d.z += (double)r.z * exp_over((double)r.m - (double)d.m, t, table);
        };
#pragma unroll
        for (int i = 0; i < 4; i++) add(p[i]);
        for (int c = lane + 128; c < chunks; c += 32) add(part[c]);
    }
    d.z = warp_sum(d.z);
    return d;
}

__device__ __forceinline__ float prob(const float* q, int x)
{
    const float v = q[x];
    return v > 0.0f ? v : 0.0f;
}

/* f(x, n, l): n of this lane's entries of [x0, x1) from x on: ends that are not
 * 16-byte aligned one by one, the rest 16 bytes at a time. */
template <typename T, typename F>
__device__ __forceinline__ void each(const T* __restrict__ row, int x0, int x1, F f)
{
    constexpr int VE = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, n = max(0, x1 - x0);
    const int head = min(n, (int)((16 - reinterpret_cast<uintptr_t>(row + x0) % 16) % 16 / sizeof(T)));
    const int nv = (n - head) / VE;
    float l[VE]; /* entries past the n are masked */
#pragma unroll
    for (int j = 1; j < VE; j++) l[j] = -INFINITY;
    if (lane < head) {
        l[0] = clean(fl_to_float(row[x0 + lane]));
        f(x0 + lane, 1, l);
    }
    const uint4* v = reinterpret_cast<const uint4*>(row + x0 + head);
#pragma unroll 2
    for (int i = lane; i < nv; i += 32) {
        const uint4 u = __ldg(v + i);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int j = 0; j < VE; j++) l[j] = clean(fl_to_float(e[j]));
        f(x0 + head + i * VE, VE, l);
    }
    const int tail = x0 + head + nv * VE + lane;
    if (tail < x1) {
#pragma unroll
        for (int j = 1; j < VE; j++) l[j] = -INFINITY;
        l[0] = clean(fl_to_float(row[tail]));
        f(tail, 1, l);
    }
}

/* This warp's sum, put beside the other warps'; the CTA's sum at its rank in
 * every CTA of the cluster, all of which have started; returns the total, the same
 * everywhere. */
__device__ __forceinline__ double share(double v, double* warps, double* ranks)
{
    namespace cg = cooperative_groups;
    const cg::cluster_group cl = cg::this_cluster();
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < kCluster) {
        double sum = 0.0;
        for (int w = 0; w < kFinWarps; w++) sum += warps[w];
        cl.map_shared_rank(ranks, threadIdx.x)[cl.block_rank()] = sum;
    }
    cl.sync();
    double all = 0.0;
    for (int r = 0; r < kCluster; r++) all += ranks[r];
    return all;
}

/* The first of n parts whose running sum exceeds the goal, else the last with
 * any weight; `before` becomes the sum of those ahead of it. */
__device__ __forceinline__ int part_of(const double* parts, int n, double goal, double& before)
{
    double run = before;
    int at = -1;
    for (int i = 0; i < n; i++) {
        if (parts[i] > 0.0) {
            at = i;
            before = run;
            if (run + parts[i] > goal) break;
        }
        run += parts[i];
    }
    return at;
}

template <typename T>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kFinThreads) verify_finish_kernel(const FlVerify g)
{
    __shared__ Decision s_row[kFinWarps];
    __shared__ int s_ok[kFinWarps];
    __shared__ double s_table[kTab], s_warps[2][kFinWarps], s_ranks[2][kCluster];
    const int s = blockIdx.x / kCluster, rank = blockIdx.x % kCluster, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = chunks_of(g.vocab);
    const RowPart* part = static_cast<const RowPart*>(g.workspace);
    const int r0 = max(g.row_start[s], 0), r1 = min(g.row_start[s + 1], g.n_rows);
    const float t = temperature_of(g, s);
    const bool greedy = !(t > 0.0f);
    const double* table = s_table;
    exp64_table(s_table);
    /* what a row's test compares; the first rows' before the wait */
    int x = -1;
    float q = 1.0f, l = -INFINITY, u = 0.0f;
    auto draft_of = [&](int row) {
        x = -1;
        if (row >= r1 - 1) return;
        x = g.draft[row];
        if (x < 0 || x >= g.vocab) x = -1;
        if (x < 0 || greedy) return;
        if (g.probs) q = prob(g.probs + row * g.probs_stride, x);
        l = clean(fl_to_float(static_cast<const T*>(g.logits)[row * g.logits_stride + x]));
        u = g.u_accept[row];
    };
    draft_of(r0 + warp);
    /* every CTA of the cluster has started before any writes into another's memory (and the table stands); under way
     * while the first kernel still runs */
    cooperative_groups::this_cluster().sync();
    fl_pdl_wait();
    if (r1 <= r0) { /* this and every later return: alike in the whole cluster */
        if (rank == 0 && threadIdx.x == 0) g.accepted[s] = 0;
        return;
    }
    /* the acceptance tests, a row per warp, in order */
    Decision d{};
    for (int base = r0;; base += kFinWarps) {
        const int row = base + warp;
        if (row < r1) {
            Decision w = merge_row(part + (size_t)row * chunks, chunks, t, table);
            w.row = row;
            bool ok = false;
            if (base > r0) draft_of(row);
            if (x >= 0 && w.m > -INFINITY)
                ok = greedy ? x == w.best : (double)u * (double)q * w.z < exp_over((double)l - (double)w.m, t, table);
            w.rej = row < r1 - 1;
            if (lane == 0) s_row[warp] = w, s_ok[warp] = ok;
        } else if (lane == 0) {
            s_ok[warp] = 1; /* behind the last row, which always stops */
        }
        __syncthreads();
        int stop = 0;
        while (stop < kFinWarps && s_ok[stop]) stop++;
        if (stop < kFinWarps) {
            d = s_row[stop];
            break;
        }
        __syncthreads();
    }
    auto write = [&](int token, int first, int step) {
        for (int row = r0 + first; row < r1; row += step)
            g.tokens[row] = row < d.row ? g.draft[row] : row == d.row ? token : -1;
        if (first == 0) g.accepted[s] = d.row - r0;
    };
    if (greedy || !(d.m > -INFINITY)) {
        if (rank == 0) write(d.m > -INFINITY ? d.best : -1, threadIdx.x, kFinThreads);
        return;
    }
    /* the sums over the row that it stopped at; this warp's entries: [x0, x1) */
    const int per = (g.vocab + kCluster * kFinWarps - 1) / (kCluster * kFinWarps);
    const int x0 = min(g.vocab, (rank * kFinWarps + warp) * per), x1 = min(g.vocab, x0 + per);
    const T* row = static_cast<const T*>(g.logits) + d.row * g.logits_stride;
    const Exp64 ew = exp64_of(d.m, t, table);
    const int skip = d.rej && !g.probs ? g.draft[d.row] : -1;
    double sum[2] = {0.0, 0.0};
    each(row, x0, x1, [&](int x, int, const float* l) {
#pragma unroll
        for (int j = 0; j < 16 / (int)sizeof(T); j++) {
            double p, scale;
            ew(x + j == skip ? -INFINITY : l[j], p, scale);
            sum[j & 1] = fma(p, scale, sum[j & 1]);
        }
    });
    const double z = share(sum[0] + sum[1], s_warps[0], s_ranks[0]);
    if (!(z > 0.0)) { /* the draft is all of p */
        if (rank == 0) write(skip, threadIdx.x, kFinThreads);
        return;
    }
    double all = z;
    const float* probs = d.rej && g.probs ? g.probs + d.row * g.probs_stride : nullptr;
    if (probs) {
        sum[0] = sum[1] = 0.0;
        each(row, x0, x1, [&](int x, int n, const float* l) {
            constexpr int VE = 16 / (int)sizeof(T);
            float p[VE] = {};
            if (n == VE && reinterpret_cast<uintptr_t>(probs + x) % 16 == 0) {
#pragma unroll
                for (int j = 0; j < VE; j += 4) {
                    const float4 v = __ldg(reinterpret_cast<const float4*>(probs + x + j));
                    p[j] = v.x, p[j + 1] = v.y, p[j + 2] = v.z, p[j + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < VE; j++)
                    if (j < n) p[j] = probs[x + j];
            }
#pragma unroll
            for (int j = 0; j < VE; j++)
                sum[j & 1] += fmax(fma((double)(p[j] > 0.0f ? -p[j] : 0.0f), z, ew.value(l[j])), 0.0);
        });
        all = share(sum[0] + sum[1], s_warps[1], s_ranks[1]);
        if (!(all > 0.0)) probs = nullptr, all = z; /* nothing is left of p - q: p itself */
    }
    /* whose range the draw falls into, and the entry in it */
    const double goal = (double)g.u_sample[s] * all;
    const int w = probs ? 1 : 0;
    double before = 0.0;
    if (part_of(s_ranks[w], kCluster, goal, before) != rank) return;
    if (part_of(s_warps[w], kFinWarps, goal, before) != warp) return;
    int token = -1;
    bool found = false;
    for (int base = x0; base < x1 && !found; base += 32 * 8) { /* eight entries of a lane, consecutive */
        const int at = base + lane * 8;
        double e[8], mine = 0.0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            e[j] = 0.0;
            if (at + j < x1 && at + j != skip) {
                e[j] = ew.value(clean(fl_to_float(row[at + j])));
                if (probs) e[j] = fmax(fma(-(double)prob(probs, at + j), z, e[j]), 0.0);
            }
            mine += e[j];
        }
        double run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        double c = before + run - mine;
        int hit = INT_MAX, last = -1;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            c += e[j];
            if (e[j] > 0.0) {
                last = at + j;
                if (c > goal && hit == INT_MAX) hit = at + j;
            }
        }
        hit = __reduce_min_sync(0xffffffffu, hit);
        last = __reduce_max_sync(0xffffffffu, last);
        found = hit != INT_MAX;
        if (found)
            token = hit;
        else if (last >= 0)
            token = last; /* rounding may leave the goal above every sum */
        before += __shfl_sync(0xffffffffu, run, 31);
    }
    write(token, lane, 32);
}

template <typename T>
cudaError_t launch(const FlVerify& v, cudaStream_t st)
{
    if (v.n_rows > 0) verify_rows_kernel<T><<<dim3(v.n_rows, chunks_of(v.vocab)), kThreads, 0, st>>>(v);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)v.n_seqs * kCluster);
    cfg.blockDim = dim3(kFinThreads);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = v.n_rows > 0 ? 1 : 0; /* with no rows the kernel before is not this call's */
    return cudaLaunchKernelEx(&cfg, verify_finish_kernel<T>, v);
}

} // namespace

size_t fl_verify_workspace_bytes(int n_rows, int, int vocab) { return (size_t)n_rows * chunks_of(vocab) * sizeof(RowPart); }

cudaError_t fl_launch_verify(const FlVerify& v, cudaStream_t st)
{
    switch (v.type) {
    case 0: return launch<float>(v, st);
    case 1: return launch<__half>(v, st);
    case 30: return launch<__nv_bfloat16>(v, st);
    default: return cudaErrorInvalidValue;
    }
}
