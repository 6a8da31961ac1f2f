/*
 * fl_paged.cuh — device helpers of the paged-cache operators: activation
 * types, the sequence and position of a packed row, cache addresses.
 */
#ifndef FL_PAGED_CUH
#define FL_PAGED_CUH

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

#endif
