/*
 * fl_paged.cuh — device helpers of the paged-cache operators: activation
 * types, the sequence and position of a packed row, cache addresses.
 */
#ifndef FL_PAGED_CUH
#define FL_PAGED_CUH

#include <climits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fl_device.cuh"
#include "fl_kernels.h"

/* Eight consecutive elements of a row as floats (16-byte aligned loads). */
__device__ __forceinline__ void fl_load8(const float* p, float (&x)[8])
{
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void fl_load8(const __half* p, float (&x)[8])
{
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void fl_load8(const __nv_bfloat16* p, float (&x)[8])
{
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void fl_store8(float* p, const float (&x)[8])
{
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void fl_store8(__half* p, const float (&x)[8])
{
    uint4 u;
    __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ void fl_store8(__nv_bfloat16* p, const float (&x)[8])
{
    uint4 u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ float fl_to_float(float x) { return x; }
__device__ __forceinline__ float fl_to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float fl_to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T fl_from_float(float x);
template <>
__device__ __forceinline__ float fl_from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half fl_from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 fl_from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

/* The sequence of packed row `row`: the last s with start[s] <= row, found by
 * the whole warp (32 starts a step, so one load for up to 32 sequences and
 * two for 1024); -1 when the row is behind the last sequence or start is not
 * in order there.  Every lane gets the result. */
__device__ __forceinline__ int fl_row_seq(const int32_t* __restrict__ start, int n_seqs, int row)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, n = n_seqs; /* the answer is in [lo, lo + n) */
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int i = lo + lane * step;
        const unsigned le = __ballot_sync(0xffffffffu, lane * step < n && __ldg(start + i) <= row);
        const int hit = le ? 31 - __clz(le) : 0;
        lo += hit * step;
        n = min(step, n - hit * step);
    }
    const int s0 = __ldg(start + lo), s1 = __ldg(start + lo + 1);
    return row >= s0 && row < s1 ? lo : -1;
}

/* Index of cache row (page, head, offset in the page) of position p of
 * sequence s, in rows of head_dim elements (and of the scale arrays); -1 when
 * the position is not mapped. */
__device__ __forceinline__ int64_t fl_cache_row(const FlPaged& c, int s, int p, int head)
{
    const int col = p >> c.page_shift;
    if (p < 0 || col >= c.cols) return -1;
    const int page = __ldg(c.table + (size_t)s * c.cols + col);
    if ((unsigned)page >= (unsigned)c.n_pages) return -1;
    return (((int64_t)page * c.n_kv + head) << c.page_shift) + (p & ((1 << c.page_shift) - 1));
}

/* ── attention helpers ── */
/* The first position that a row at position p (down to -n_rows: the host bounds the window by that) sees. */
__device__ __forceinline__ int fl_first_seen(int p, int window) { return window > 0 ? max(p + 1 - window, 0) : 0; }
/* A sequence's length, kept where a tile from its last position on is in range; no table reaches further. */
__device__ __forceinline__ int fl_seq_len(const FlPaged& c, int s) { return min(max(__ldg(c.seq_len + s), 0), INT_MAX - 4096); }
__device__ __forceinline__ float fl_ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
/* x * 2^e for any e that a float's exponent range may ask for, in two exact steps. */
__device__ __forceinline__ float fl_pow2(int e) { return __int_as_float((e + 127) << 23); } /* e in [-126, 127] */
__device__ __forceinline__ float fl_scale2(float x, int e)
{
    const int h = e >> 1;
    return x * fl_pow2(h) * fl_pow2(e - h);
}
__device__ __forceinline__ uint32_t fl_half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ uint32_t fl_pack_half2(float a, float b) { return fl_half2_bits(__floats2half2_rn(a, b)); }

/* n / grp by the host's reciprocal floor(2^64 / grp) + 1 (0 for grp = 1). */
__device__ __forceinline__ int fl_div_grp(const FlPagedAttn& a, int n)
{
    return a.grp_inv ? (int)__umul64hi((unsigned long long)(uint32_t)n, a.grp_inv) : n;
}

/* The four 8-bit elements of w as halves, exactly: bytes 0, 1 in lo, 2, 3 in hi. */
template <int KV>
__device__ __forceinline__ void fl_widen4(uint32_t w, uint32_t& lo, uint32_t& hi)
{
    if constexpr (KV == FL_KV_Q8) {
        /* 0x6400 + u is the half 1024 + u; u = q + 128 */
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        lo = fl_half2_bits(__hsub2(*reinterpret_cast<const __half2*>(&a), bias));
        hi = fl_half2_bits(__hsub2(*reinterpret_cast<const __half2*>(&b), bias));
    } else {
        const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
        const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
        lo = (uint32_t)a.x | ((uint32_t)a.y << 16);
        hi = (uint32_t)b.x | ((uint32_t)b.y << 16);
    }
}

__device__ __forceinline__ void fl_cp_async16(uint32_t dst, const void* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void fl_cp_async8(uint32_t dst, const void* src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void fl_cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fl_cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

/* The schedule of an attention kernel: units [c * per, (c + 1) * per) are CTA
 * c's range.  All below 2^32, which the host has checked on the largest
 * possible total. */
constexpr int kFlWaitCtas = 148; /* CTAs at most of the kernel that has waits */
struct FlSchedule {
    uint32_t total, per;
    alignas(4) uint8_t expired[kFlWaitCtas]; /* whether a wait of the CTA ran out */
};
static_assert(sizeof(FlSchedule) <= 256, "its place in the workspace");

/* Workspace: the schedule, the first unit of each sequence, then the partials'
 * (m, l) and outputs in two slots of `rows` rows per CTA: [2c] for a range that
 * continues an item, [2c + 1] for one that starts it. */
struct FlAttnSpace {
    FlSchedule* sched;
    uint32_t* seq_unit;
    float2* ml;
    float* o;
};
__host__ __device__ __forceinline__ size_t fl_align256(size_t b) { return (b + 255) & ~(size_t)255; }
__host__ __device__ __forceinline__ FlAttnSpace fl_attn_space(void* p, int n_seqs, int ctas, int rows, int hd,
                                                              size_t* bytes = nullptr)
{
    uint8_t* b = static_cast<uint8_t*>(p);
    FlAttnSpace w;
    size_t at = 256;
    w.sched = reinterpret_cast<FlSchedule*>(b);
    w.seq_unit = reinterpret_cast<uint32_t*>(b + at);
    at += fl_align256((size_t)n_seqs * 4);
    w.ml = reinterpret_cast<float2*>(b + at);
    at += fl_align256((size_t)2 * ctas * rows * 8);
    w.o = reinterpret_cast<float*>(b + at);
    at += (size_t)2 * ctas * rows * hd * 4;
    if (bytes) *bytes = at;
    return w;
}

/* The output of one (row, head) that a wait ran out on: no number, and counted, by a warp. */
template <typename T, int HD>
__device__ __forceinline__ void fl_nan_row(const FlPagedAttn& a, int row, int h)
{
    const float nan = __uint_as_float(0x7fffffffu);
    const int lane = threadIdx.x & 31;
    T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_stride + (int64_t)h * HD;
    for (int e = lane; e < HD; e += 32) out[e] = fl_from_float<T>(nan);
    if (a.lse && lane == 0) a.lse[(int64_t)row * a.n_heads + h] = nan;
    if (lane == 0) atomicAdd(a.expired, 1u);
}

/* The output of one (row, head) whose item ranges c0 .. c1 share, its row r of
 * `rows`: one warp adds the partials in range order; a lane holds one partial's
 * weight, and HD / 32 elements. */
template <typename T, int HD>
__device__ __forceinline__ void fl_merge_row(const FlPagedAttn& a, const FlAttnSpace& ws, int c0, int c1, int r, int rows,
                                             int row, int h)
{
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 31;
    float M = -INFINITY, L = 0.0f, o[E] = {};
    for (int base = c0; base <= c1; base += 32) {
        const int i = base + lane, n = min(32, c1 - base + 1);
        const float2 ml = i <= c1 ? ws.ml[(2 * i + (i == c0)) * rows + r] : make_float2(-INFINITY, 0.0f);
        const float mx = fmaxf(M, fl_warp_max(ml.x));
        if (mx > M) {
            const float f0 = fl_ex2(M - mx); /* 0 the first time */
            L *= f0;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] *= f0;
            M = mx;
        }
        const float w = ml.x == -INFINITY ? 0.0f : fl_ex2(ml.x - M);
        L += fl_warp_sum(ml.x == -INFINITY ? ml.y : ml.y * w); /* a NaN sum stays one */
#pragma unroll 4
        for (int j = 0; j < n; j++) {
            const int at = 2 * (base + j) + (base + j == c0);
            const float wj = __shfl_sync(0xffffffffu, w, j);
            const float* src = ws.o + ((size_t)at * rows + r) * HD + lane * E;
            if constexpr (E == 2) {
                const float2 u = *reinterpret_cast<const float2*>(src);
                o[0] = fmaf(u.x, wj, o[0]), o[1] = fmaf(u.y, wj, o[1]);
            } else {
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    const float4 u = *reinterpret_cast<const float4*>(src + e);
                    o[e] = fmaf(u.x, wj, o[e]), o[e + 1] = fmaf(u.y, wj, o[e + 1]);
                    o[e + 2] = fmaf(u.z, wj, o[e + 2]), o[e + 3] = fmaf(u.w, wj, o[e + 3]);
                }
            }
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_stride + (int64_t)h * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) out[e] = fl_from_float<T>(o[e] * inv);
    if (a.lse && lane == 0) a.lse[(int64_t)row * a.n_heads + h] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.693147181f;
}

#endif
