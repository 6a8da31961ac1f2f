/*
 * fl_verify.cu — verification of drafted tokens against the target's logits
 * (fl_verify_device).
 *
 * Bound by reading the logits once; four kernels, each started early and
 * waiting for the one before (programmatic dependent launch), over chunks of
 * 4096 vocabulary entries so that one sequence and sixty-four both spread over
 * the SMs:
 *  rows: per (row, chunk) the maximum with its first index and the sum of
 *        exp((l - max) / T), exponentials in fp32;
 *  stop: per (sequence, chunk) first the acceptance tests, which every chunk's
 *        CTA repeats (a few rows of a few partials), then the chunk's sum over
 *        the row that the sequence stopped at, exponentials and sums in 64 bits;
 *  rest: the same for max(p - q, 0), which needs that sum's total first;
 *  draw: per sequence the chunk that the draw falls into, and the entry in it.
 * The draw compares with cumulative sums of up to 2^24 entries, whose borders
 * lie closer than fp32 resolves, hence the 64 bits there; the acceptance tests
 * compare single probabilities, for which the fp32 exponentials' 2^-22 is
 * enough.
 */
#include <cfloat>
#include <climits>

#include "fl_paged.cuh"

namespace {

constexpr int kThreads = 128, kStopThreads = 256, kChunk = 4096;
constexpr int kDrawThreads = 512;

struct RowPart { /* of a row's chunk */
    float m, z;
    int32_t best, pad;
};
struct Decision { /* of a sequence */
    double z;    /* sum of exp((l - m) / T) over the row, exponentials in fp32 */
    float m;
    int32_t row; /* that it stopped at; -1: no rows */
    int32_t rej, best;
};
struct Sums { /* of a chunk of that row */
    double e;    /* of exp((l - m) / T), less the draft's where it was rejected and certain */
    double rest; /* of max(exp - q Z, 0) */
};

struct Space {
    RowPart* part;   /* [n_rows][chunks] */
    Decision* dec;   /* [n_seqs] */
    Sums* sums;      /* [n_seqs][chunks] */
};
__host__ __device__ __forceinline__ int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }
__host__ __device__ __forceinline__ Space space(void* p, int n_rows, int n_seqs, int vocab, size_t* bytes = nullptr)
{
    uint8_t* b = static_cast<uint8_t*>(p);
    const size_t c = (size_t)chunks_of(vocab);
    Space s;
    size_t at = 0;
    s.part = reinterpret_cast<RowPart*>(b);
    at += fl_align256(n_rows * c * sizeof(RowPart));
    s.dec = reinterpret_cast<Decision*>(b + at);
    at += fl_align256(n_seqs * sizeof(Decision));
    s.sums = reinterpret_cast<Sums*>(b + at);
    at += n_seqs * c * sizeof(Sums);
    if (bytes) *bytes = at;
    return s;
}

/* NaN is masked, +infinity is the largest finite value. */
__device__ __forceinline__ float clean(float l) { return l != l ? -INFINITY : fminf(l, FLT_MAX); }

/* e^((l - m) / T) in 64 bits as 2^(k / 32), k = (l - m) A with A = 32 log2(e) /
 * T: k = n + f, |f| <= 1/2; 2^(n / 32) from a table of 32 and an exponent,
 * 2^(f / 32) by its Taylor series to f^5 (the next term is below 2^-48). */
constexpr double kL = 0.69314718055994531 / 32.0;
struct Exp64 {
    double a, m;
    const double* table; /* 2^(i / 32), i < 32, in shared memory */
    __device__ __forceinline__ double operator()(float l) const
    {
        const double k = ((double)l - m) * a;
        if (!(k > -32.0 * 1021.0)) return 0.0; /* below 2^-1021; masked */
        const double magic = 6755399441055744.0; /* 1.5 * 2^52: the sum's low word is k rounded */
        const double t = k + magic;
        const int n = __double2loint(t);
        const double f = k - (t - magic);
        double p = kL * kL * kL * kL * kL / 120.0;
        p = fma(p, f, kL * kL * kL * kL / 24.0);
        p = fma(p, f, kL * kL * kL / 6.0);
        p = fma(p, f, kL * kL / 2.0);
        p = fma(p, f, kL);
        p = fma(p, f, 1.0);
        p *= table[n & 31];
        return __hiloint2double(__double2hiint(p) + ((n >> 5) << 20), __double2loint(p));
    }
};
__device__ __forceinline__ void exp64_table(double* table)
{
    if (threadIdx.x < 32) {
        /* e^(i kL) by its series; i kL < 0.7 */
        const double y = kL * (double)(int)threadIdx.x;
        double p = 1.0;
        for (int i = 20; i > 0; i--) p = fma(p, y / (double)i, 1.0);
        table[threadIdx.x] = p;
    }
}
__device__ __forceinline__ Exp64 exp64_of(float m, float t, const double* table)
{
    return Exp64{46.166241308446828 / (double)t, (double)m, table}; /* 32 log2(e) */
}

__device__ __forceinline__ double warp_sum(double v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

/* f(x, n, l): n of this thread's entries of [x0, x1) from x on, by threads and
 * ascending: ends that are not 16-byte aligned one by one, the rest 16 bytes
 * at a time. */
template <int NT, typename T, typename F>
__device__ __forceinline__ void each(const T* __restrict__ row, int x0, int x1, F f)
{
    constexpr int VE = 16 / sizeof(T);
    const int n = x1 - x0;
    const int head = min(n, (int)((16 - reinterpret_cast<uintptr_t>(row + x0) % 16) % 16 / sizeof(T)));
    const int nv = (n - head) / VE;
    float l[VE] = {};
    if ((int)threadIdx.x < head) {
        l[0] = clean(fl_to_float(row[x0 + threadIdx.x]));
        f(x0 + (int)threadIdx.x, 1, l);
    }
    const uint4* v = reinterpret_cast<const uint4*>(row + x0 + head);
#pragma unroll 2
    for (int i = threadIdx.x; i < nv; i += NT) {
        const uint4 u = __ldg(v + i);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int j = 0; j < VE; j++) l[j] = clean(fl_to_float(e[j]));
        f(x0 + head + i * VE, VE, l);
    }
    const int tail = x0 + head + nv * VE + threadIdx.x;
    if (tail < x1) {
        l[0] = clean(fl_to_float(row[tail]));
        f(tail, 1, l);
    }
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
    float z = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            z += fl_ex2((__uint_as_float(w[i]) - m) * c);
        } else {
            const float2 f = halves(w[i], T());
            z += fl_ex2((f.x - m) * c) + fl_ex2((f.y - m) * c);
        }
    }
    return z;
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
    const float t = g.temperature[s];
    float m = fmaxf(ends[0], ends[1]);
#pragma unroll
    for (int i = 0; i < NV; i++)
        if ((int)threadIdx.x + i * kThreads < nv) m = fmaxf(m, max_of<T>(u[i]));
    m = fminf(m, FLT_MAX);
    const float mine = m;
    m = fl_warp_max(m);
    /* its first index, looked for by the threads that hold it */
    int best = INT_MAX;
    if (mine == m && m > -INFINITY) {
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
        const Space sp = space(g.workspace, g.n_rows, g.n_seqs, g.vocab);
        sp.part[(size_t)row * gridDim.y + chunk] = RowPart{M, Z, B, 0};
    }
}

/* A row's maximum, first index of it and sum, by a warp from its chunks: up to
 * 128 of them are loaded at once, more a second time. */
__device__ __forceinline__ Decision merge_row(const RowPart* __restrict__ part, int chunks, float t, const double* table)
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
        const Exp64 e = exp64_of(d.m, t, table);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (p[i].m > -INFINITY) d.z += (double)p[i].z * e(p[i].m);
        for (int c = lane + 128; c < chunks; c += 32)
            if (part[c].m > -INFINITY) d.z += (double)part[c].z * e(part[c].m);
    }
    d.z = warp_sum(d.z);
    return d;
}

__device__ __forceinline__ float prob(const float* q, int x)
{
    const float v = q[x];
    return v > 0.0f ? v : 0.0f;
}

template <typename T>
__global__ void __launch_bounds__(kStopThreads) verify_stop_kernel(const FlVerify g)
{
    __shared__ Decision s_row[kStopThreads / 32];
    __shared__ int s_ok[kStopThreads / 32];
    __shared__ double s_d[kStopThreads / 32], s_table[32];
    const int chunk = blockIdx.y, s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, chunks = gridDim.y;
    fl_pdl_trigger();
    const Space sp = space(g.workspace, g.n_rows, g.n_seqs, g.vocab);
    const int r0 = max(g.row_start[s], 0), r1 = min(g.row_start[s + 1], g.n_rows);
    const float t = g.temperature[s];
    const bool greedy = !(t > 0.0f);
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
    __syncthreads();
    fl_pdl_wait();
    if (r1 <= r0) {
        if (chunk == 0 && threadIdx.x == 0) sp.dec[s] = Decision{0.0, -INFINITY, -1, 0, -1};
        return;
    }
    /* the acceptance tests, a row per warp, in order */
    Decision d{};
    for (int base = r0;; base += kStopThreads / 32) {
        const int row = base + warp;
        if (row < r1) {
            Decision w = merge_row(sp.part + (size_t)row * chunks, chunks, t, s_table);
            w.row = row;
            bool ok = false;
            if (base > r0) draft_of(row);
            if (x >= 0 && w.m > -INFINITY)
                ok = greedy ? x == w.best : (double)u * (double)q * w.z < exp64_of(w.m, t, s_table)(l);
            w.rej = row < r1 - 1;
            if (lane == 0) s_row[warp] = w, s_ok[warp] = ok;
        } else if (lane == 0) {
            s_ok[warp] = 1; /* behind the last row, which always stops */
        }
        __syncthreads();
        int stop = 0;
        while (stop < kStopThreads / 32 && s_ok[stop]) stop++;
        if (stop < kStopThreads / 32) {
            d = s_row[stop];
            break;
        }
        __syncthreads();
    }
    if (chunk == 0 && threadIdx.x == 0) sp.dec[s] = d;
    if (greedy || !(d.m > -INFINITY)) return;
    /* the chunk's sum over the row that it stopped at */
    const int skip = d.rej && !g.probs ? g.draft[d.row] : -1;
    const Exp64 ew = exp64_of(d.m, t, s_table);
    double sum = 0.0;
    each<kStopThreads>(static_cast<const T*>(g.logits) + d.row * g.logits_stride, chunk * kChunk, min(g.vocab, (chunk + 1) * kChunk),
         [&](int x, int n, const float* l) {
#pragma unroll
             for (int j = 0; j < 16 / (int)sizeof(T); j++)
                 if (j < n && x + j != skip) sum += ew(l[j]);
         });
    sum = warp_sum(sum);
    if (lane == 0) s_d[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kStopThreads / 32; w++) sum += s_d[w];
        sp.sums[(size_t)s * chunks + chunk].e = sum;
    }
}

/* The sum of a sequence's chunks, the same in every thread of a warp. */
template <bool REST>
__device__ __forceinline__ double total_of(const Sums* __restrict__ s, int chunks)
{
    double v = 0.0;
    for (int c = threadIdx.x & 31; c < chunks; c += 32) v += REST ? s[c].rest : s[c].e;
    return warp_sum(v);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_rest_kernel(const FlVerify g)
{
    __shared__ double s_d[kThreads / 32], s_table[32];
    const int chunk = blockIdx.y, s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, chunks = gridDim.y;
    fl_pdl_trigger();
    const Space sp = space(g.workspace, g.n_rows, g.n_seqs, g.vocab);
    const float t = g.temperature[s];
    exp64_table(s_table);
    __syncthreads();
    fl_pdl_wait();
    const Decision d = sp.dec[s];
    if (d.row < 0 || !d.rej || !(t > 0.0f) || !(d.m > -INFINITY)) return;
    const double z = total_of<false>(sp.sums + (size_t)s * chunks, chunks);
    const Exp64 ew = exp64_of(d.m, t, s_table);
    const float* q = g.probs + d.row * g.probs_stride;
    double sum = 0.0;
    each<kThreads>(static_cast<const T*>(g.logits) + d.row * g.logits_stride, chunk * kChunk,
                   min(g.vocab, (chunk + 1) * kChunk), [&](int x, int n, const float* l) {
             constexpr int VE = 16 / (int)sizeof(T);
             float p[VE] = {};
             if (n == VE && reinterpret_cast<uintptr_t>(q + x) % 16 == 0) {
#pragma unroll
                 for (int j = 0; j < VE; j += 4) {
                     const float4 v = __ldg(reinterpret_cast<const float4*>(q + x + j));
                     p[j] = v.x, p[j + 1] = v.y, p[j + 2] = v.z, p[j + 3] = v.w;
                 }
             } else {
#pragma unroll
                 for (int j = 0; j < VE; j++)
                     if (j < n) p[j] = q[x + j];
             }
#pragma unroll
             for (int j = 0; j < VE; j++)
                 if (j < n) sum += fmax(ew(l[j]) - (double)(p[j] > 0.0f ? p[j] : 0.0f) * z, 0.0);
         });
    sum = warp_sum(sum);
    if (lane == 0) s_d[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 32; w++) sum += s_d[w];
        sp.sums[(size_t)s * chunks + chunk].rest = sum;
    }
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads) verify_draw_kernel(const FlVerify g)
{
    constexpr int PER = kChunk / kDrawThreads; /* consecutive entries of a thread */
    __shared__ double s_w[kDrawThreads / 32], s_table[32];
    __shared__ double s_before;
    __shared__ int s_chunk, s_tok, s_last;
    const int s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, chunks = chunks_of(g.vocab);
    const Space sp = space(g.workspace, g.n_rows, g.n_seqs, g.vocab);
    const int r0 = max(g.row_start[s], 0), r1 = min(g.row_start[s + 1], g.n_rows);
    const float t = g.temperature[s];
    exp64_table(s_table);
    __syncthreads();
    fl_pdl_wait();
    const Decision d = sp.dec[s];
    if (d.row < 0) {
        if (threadIdx.x == 0) g.accepted[s] = 0;
        return;
    }
    int token = -1;
    const Sums* sums = sp.sums + (size_t)s * chunks;
    const bool greedy = !(t > 0.0f);
    const double z = greedy || !(d.m > -INFINITY) ? 0.0 : total_of<false>(sums, chunks);
    const int skip = d.rej && !g.probs ? g.draft[d.row] : -1;
    if (d.m > -INFINITY && greedy) {
        token = d.best;
    } else if (d.m > -INFINITY && !(z > 0.0)) {
        token = skip; /* the draft is all of p */
    } else if (d.m > -INFINITY) {
        const Exp64 ew = exp64_of(d.m, t, s_table);
        bool rest = d.rej && g.probs;
        double all = z;
        if (rest) {
            all = total_of<true>(sums, chunks);
            if (!(all > 0.0)) rest = false, all = z; /* nothing is left of p - q: p itself */
        }
        const double goal = (double)g.u_sample[s] * all;
        /* the first chunk whose running sum exceeds the goal; else the last that has any weight */
        if (warp == 0) {
            double before = 0.0, before_last = 0.0;
            int hit = -1, last = 0;
            for (int c0 = 0; c0 < chunks && hit < 0; c0 += 32) {
                const int c = c0 + lane;
                const double w = c < chunks ? (rest ? sums[c].rest : sums[c].e) : 0.0;
                double run = w;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double u = __shfl_up_sync(0xffffffffu, run, o);
                    if (lane >= o) run += u;
                }
                const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
                const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && before + run > goal);
                const int at = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : -1;
                if (at >= 0) {
                    last = c0 + at;
                    before_last = before + __shfl_sync(0xffffffffu, run - w, at);
                }
                if (over) hit = last;
                before += __shfl_sync(0xffffffffu, run, 31);
            }
            if (lane == 0) s_chunk = last, s_before = before_last, s_tok = INT_MAX, s_last = -1;
        }
        __syncthreads();
        /* the entry in it */
        const int x0 = s_chunk * kChunk + threadIdx.x * PER;
        const T* l = static_cast<const T*>(g.logits) + d.row * g.logits_stride;
        const float* q = rest ? g.probs + d.row * g.probs_stride : nullptr;
        double w[PER], mine = 0.0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int x = x0 + i;
            w[i] = 0.0;
            if (x < g.vocab && x != skip) {
                w[i] = ew(clean(fl_to_float(l[x])));
                if (rest) w[i] = fmax(w[i] - (double)prob(q, x) * z, 0.0);
            }
            mine += w[i];
        }
        double run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double u = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += u;
        }
        if (lane == 31) s_w[warp] = run;
        __syncthreads();
        double c = s_before + run - mine;
        for (int i = 0; i < warp; i++) c += s_w[i];
        int last = -1, hit = INT_MAX;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            c += w[i];
            if (w[i] > 0.0) {
                last = x0 + i;
                if (c > goal && hit == INT_MAX) hit = x0 + i;
            }
        }
        if (hit != INT_MAX) atomicMin(&s_tok, hit);
        if (last >= 0) atomicMax(&s_last, last);
        __syncthreads();
        token = s_tok != INT_MAX ? s_tok : s_last;
    }
    for (int row = r0 + threadIdx.x; row < r1; row += kDrawThreads)
        g.tokens[row] = row < d.row ? g.draft[row] : row == d.row ? token : -1;
    if (threadIdx.x == 0) g.accepted[s] = d.row - r0;
}

template <typename K>
cudaError_t after(K kernel, dim3 grid, int threads, const FlVerify& v, cudaStream_t st)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, v);
}

template <typename T>
cudaError_t launch(const FlVerify& v, cudaStream_t st)
{
    const unsigned chunks = chunks_of(v.vocab);
    if (v.n_rows > 0) verify_rows_kernel<T><<<dim3(v.n_rows, chunks), kThreads, 0, st>>>(v);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = after(verify_stop_kernel<T>, dim3(v.n_seqs, chunks), kStopThreads, v, st);
    if (e == cudaSuccess && v.probs) e = after(verify_rest_kernel<T>, dim3(v.n_seqs, chunks), kThreads, v, st);
    if (e == cudaSuccess) e = after(verify_draw_kernel<T>, dim3(v.n_seqs), kDrawThreads, v, st);
    return e;
}

} // namespace

size_t fl_verify_workspace_bytes(int n_rows, int n_seqs, int vocab)
{
    size_t bytes;
    space(nullptr, n_rows, n_seqs, vocab, &bytes);
    return bytes;
}

cudaError_t fl_launch_verify(const FlVerify& v, cudaStream_t st)
{
    switch (v.type) {
    case 0: return launch<float>(v, st);
    case 1: return launch<__half>(v, st);
    case 30: return launch<__nv_bfloat16>(v, st);
    default: return cudaErrorInvalidValue;
    }
}
