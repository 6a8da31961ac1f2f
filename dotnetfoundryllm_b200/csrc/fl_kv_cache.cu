/*
 * fl_kv_cache.cu — append to and gather from a paged KV cache
 * (fl_kv_append_device, fl_kv_gather_device).
 *
 * Work: (row, kv head) pairs, K and V together.  A pair's head_dim elements
 * are spread over head_dim / 8 lanes, eight each (one or two 16-byte loads),
 * so that a row's maximum is a few shuffles and every access is a full
 * sector; a warp holds 32 / (head_dim / 8) pairs.  Both directions are one
 * pass: every element read once and written once.
 */
#include "fl_paged.cuh"

namespace {

constexpr int kThreads = 256;

/* Eight quotients x / s rounded to the nearest integer, ties to even, as bytes.
 * x * (1/s) is off by a few ulp at most, so the rounded candidate can only be
 * wrong next to a border k + 1/2: the remainder x - q s is exact in one FMA (a
 * multiple of the smaller ulp, at most about s/2), and where it reaches s/2,
 * which is rare, it decides.  Adding 1.5 2^23 rounds, and leaves the byte in the
 * low bits: no conversion instructions, whose rate bound the kernel.  |x| is at
 * most 127 s (1 + 2^-24), which rounds to 127. */
__device__ __forceinline__ uint2 quant_q8(const float (&x)[8], float s, float inv)
{
    constexpr float kMagic = 12582912.0f;
    const float h = 0.5f * s;
    float t[8];
    bool near = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        t[i] = fmaf(x[i], inv, kMagic);
        near |= fabsf(fmaf(kMagic - t[i], s, x[i])) >= h;
    }
    if (near) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float q = t[i] - kMagic;
            const float r = fmaf(-q, s, x[i]);
            if (fabsf(r) > h || (fabsf(r) == h && ((int)q & 1))) q += r > 0.0f ? 1.0f : -1.0f;
            t[i] = q + kMagic;
        }
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        w[i] = __byte_perm(__byte_perm(__float_as_uint(t[4 * i]), __float_as_uint(t[4 * i + 1]), 0x0040),
                           __byte_perm(__float_as_uint(t[4 * i + 2]), __float_as_uint(t[4 * i + 3]), 0x0040), 0x5410);
    return make_uint2(w[0], w[1]);
}

/* Eight numbers as e4m3 bytes. */
__device__ __forceinline__ uint2 pack_f8(const float (&y)[8])
{
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[4 * i], y[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
               (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[4 * i + 2], y[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16;
    return make_uint2(w[0], w[1]);
}

/* Eight quotients x / s rounded to e4m3 as the exact quotients round.  x * (1/s)
 * is within 2 ulp of the quotient, so where 4 ulp (2^-21) less and 4 ulp more of
 * it round alike, the quotient does too.  Elsewhere, which is rare, a border
 * between e4m3 values lies in between: a number t of at most 5 significant bits.
 * The sign of x - t s (one FMA, exact in sign) tells on which side of t the
 * quotient lies, and t or its neighbour stands for it. */
__device__ __forceinline__ uint2 quant_f8(const float (&x)[8], float s, float inv)
{
    float y[8];
    const float lo = fmaf(inv, -4.7683716e-7f, inv), hi = fmaf(inv, 4.7683716e-7f, inv);
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = x[i] * lo;
    const uint2 a = pack_f8(y);
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = x[i] * hi;
    const uint2 b = pack_f8(y);
    if (((a.x ^ b.x) | (a.y ^ b.y)) == 0) return a;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        y[i] = x[i] * inv;
        const uint32_t b = __float_as_uint(y[i]), t = (b + (1u << 18)) & ~((1u << 19) - 1u); /* 4 fraction bits */
        const int d = (int)(b - t);
        /* below 2^-12 everything rounds to 0: half the smallest value is 2^-10 */
        if (d > 16 || d < -16 || fabsf(y[i]) < 2.4414062e-4f) continue;
        const float tf = __uint_as_float(t), r = fmaf(-tf, s, x[i]);
        y[i] = r == 0.0f ? tf : __uint_as_float((r > 0.0f) == (tf > 0.0f) ? t + 1u : t - 1u);
    }
    return pack_f8(y);
}

template <int KV>
struct Packed8 { /* eight elements in the cache */
    uint2 w;
};
template <>
struct Packed8<FL_KV_F16> {
    uint4 w;
};

/* Eight elements of a row and the row's scale; `lanes` consecutive lanes hold the row. */
template <int KV, int LANES>
__device__ __forceinline__ Packed8<KV> quantize8(const float (&x)[8], float& scale)
{
    Packed8<KV> out;
    if constexpr (KV == FL_KV_F16) {
        __half2* h = reinterpret_cast<__half2*>(&out.w);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float f = x[2 * i + j];
                v[j] = fabsf(f) > 65504.0f ? copysignf(65504.0f, f) : f; /* NaN stays */
            }
            h[i] = __floats2half2_rn(v[0], v[1]);
        }
    } else {
        /* the maximum magnitude by integer compares: NaN above infinity above every number */
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) a = max(a, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
        const bool finite = a < 0x7f800000u;
        constexpr float top = KV == FL_KV_Q8 ? 127.0f : 448.0f;
        const float s = finite ? __fdiv_rn(__uint_as_float(a), top) : __uint_as_float(0x7fffffffu);
        scale = s;
        out.w = make_uint2(0, 0);
        if (s >= 7.8886091e-31f) { /* 2^-100; false for NaN */
            out.w = KV == FL_KV_Q8 ? quant_q8(x, s, __fdiv_rn(1.0f, s)) : quant_f8(x, s, __fdiv_rn(1.0f, s));
        } else if (s > 0.0f) {
            /* scaled up with its row, so that its reciprocal is finite; a subnormal scale is rounded to a whole number of
             * 2^-149, so that quotients may pass the largest code by any factor below 2: they are cut to it */
            float y[8];
            const float su = s * 1.2676506e30f, most = top * su; /* 2^100 */
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = fminf(fmaxf(x[i] * 1.2676506e30f, -most), most);
            out.w = KV == FL_KV_Q8 ? quant_q8(y, su, __fdiv_rn(1.0f, su)) : quant_f8(y, su, __fdiv_rn(1.0f, su));
        }
    }
    return out;
}

template <int KV>
__device__ __forceinline__ void dequantize8(const Packed8<KV>& p, float s, float (&x)[8])
{
    if constexpr (KV == FL_KV_F16) {
        const __half2* h = reinterpret_cast<const __half2*>(&p.w);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    } else {
        const uint32_t w[2] = {p.w.x, p.w.y};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            uint32_t h[2];
            fl_widen4<KV>(w[i], h[0], h[1]);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
                x[4 * i + 2 * j] = f.x * s, x[4 * i + 2 * j + 1] = f.y * s;
            }
        }
    }
}

template <int KV>
__device__ __forceinline__ void store_cache(const FlPaged& c, bool v, int64_t at, int e, const Packed8<KV>& p, float s)
{
    constexpr int ES = KV == FL_KV_F16 ? 2 : 1;
    uint8_t* base = static_cast<uint8_t*>(v ? c.v : c.k) + (at * c.hd + e) * ES;
    if constexpr (KV == FL_KV_F16) {
        *reinterpret_cast<uint4*>(base) = p.w;
    } else {
        *reinterpret_cast<uint2*>(base) = p.w;
        if (e == 0) (v ? c.v_scale : c.k_scale)[at] = s;
    }
}

template <typename T, int KV, int HD>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const FlPaged c, const T* __restrict__ k, int64_t k_stride,
                                                             const T* __restrict__ v, int64_t v_stride)
{
    constexpr int LANES = HD / 8, PER_WARP = 32 / LANES;
    const int lane = threadIdx.x & 31, e = (lane % LANES) * 8;
    const int64_t warp = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
    const int64_t pair0 = warp * PER_WARP, n_pairs = (int64_t)c.n_rows * c.n_kv;
    if (pair0 >= n_pairs) return;
    const int mine = lane / LANES;
    /* the rows, under way while their places are looked up */
    float xk[8], xv[8];
    {
        const int64_t pair = min(pair0 + mine, n_pairs - 1);
        const int row = (int)((uint32_t)pair / (uint32_t)c.n_kv), head = (int)(pair - (int64_t)row * c.n_kv);
        fl_load8(k + row * k_stride + head * HD + e, xk);
        fl_load8(v + row * v_stride + head * HD + e, xv);
    }
    /* each pair's place; consecutive pairs are mostly heads of one row */
    int prev = -1, s = -1;
    int64_t my_at = -1;
#pragma unroll
    for (int i = 0; i < PER_WARP; i++) {
        const int64_t pair = pair0 + i;
        if (pair < n_pairs) {
            const int row = (int)((uint32_t)pair / (uint32_t)c.n_kv), head = (int)(pair - (int64_t)row * c.n_kv);
            if (row != prev) s = fl_row_seq(c.row_start, c.n_seqs, row);
            prev = row;
            if (s >= 0 && i == mine)
                my_at = fl_cache_row(c, s, __ldg(c.seq_len + s) - (__ldg(c.row_start + s + 1) - row), head);
        }
    }
    float sk = 0.0f, sv = 0.0f;
    const Packed8<KV> pk = quantize8<KV, LANES>(xk, sk), pv = quantize8<KV, LANES>(xv, sv);
    if (my_at >= 0) {
        store_cache<KV>(c, false, my_at, e, pk, sk);
        store_cache<KV>(c, true, my_at, e, pv, sv);
    }
}

template <typename T, int KV, int HD>
__global__ void __launch_bounds__(kThreads) kv_gather_kernel(const FlPaged c, T* __restrict__ k, int64_t k_stride,
                                                             T* __restrict__ v, int64_t v_stride)
{
    constexpr int LANES = HD / 8, PER_WARP = 32 / LANES, ES = KV == FL_KV_F16 ? 2 : 1;
    const int lane = threadIdx.x & 31, e = (lane % LANES) * 8;
    const int64_t warp = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
    const int64_t pair0 = warp * PER_WARP, n_pairs = (int64_t)c.n_rows * c.n_kv;
    if (pair0 >= n_pairs) return;
    const int mine = lane / LANES;
    int prev = -1, s = -1, my_s = -1;
#pragma unroll
    for (int i = 0; i < PER_WARP; i++) {
        const int64_t pair = pair0 + i;
        if (pair < n_pairs) {
            const int row = (int)(pair / c.n_kv);
            if (row != prev) s = fl_row_seq(c.row_start, c.n_seqs, row);
            prev = row;
            if (i == mine) my_s = s;
        }
    }
    if (my_s < 0) return;
    const int64_t pair = pair0 + mine;
    const int row = (int)(pair / c.n_kv), head = (int)(pair - (int64_t)row * c.n_kv);
    const int64_t at = fl_cache_row(c, my_s, __ldg(c.seq_len + my_s) - (__ldg(c.row_start + my_s + 1) - row), head);
    float xk[8] = {}, xv[8] = {};
    if (at >= 0) {
        Packed8<KV> pk, pv;
        const uint8_t* kb = static_cast<const uint8_t*>(c.k) + (at * HD + e) * ES;
        const uint8_t* vb = static_cast<const uint8_t*>(c.v) + (at * HD + e) * ES;
        float sk = 1.0f, sv = 1.0f;
        if constexpr (KV == FL_KV_F16) {
            pk.w = *reinterpret_cast<const uint4*>(kb);
            pv.w = *reinterpret_cast<const uint4*>(vb);
        } else {
            pk.w = *reinterpret_cast<const uint2*>(kb);
            pv.w = *reinterpret_cast<const uint2*>(vb);
            sk = c.k_scale[at];
            sv = c.v_scale[at];
        }
        dequantize8<KV>(pk, sk, xk);
        dequantize8<KV>(pv, sv, xv);
    }
    fl_store8(k + row * k_stride + head * HD + e, xk);
    fl_store8(v + row * v_stride + head * HD + e, xv);
}

template <typename T, int KV, int HD>
cudaError_t launch(bool append, const FlPaged& c, void* k, int64_t ks, void* v, int64_t vs, cudaStream_t st)
{
    const int64_t pairs = (int64_t)c.n_rows * c.n_kv, per_block = (int64_t)(kThreads / 32) * (256 / HD);
    const unsigned grid = (unsigned)((pairs + per_block - 1) / per_block);
    if (append)
        kv_append_kernel<T, KV, HD><<<grid, kThreads, 0, st>>>(c, static_cast<const T*>(k), ks,
                                                               static_cast<const T*>(v), vs);
    else
        kv_gather_kernel<T, KV, HD><<<grid, kThreads, 0, st>>>(c, static_cast<T*>(k), ks, static_cast<T*>(v), vs);
    return cudaGetLastError();
}

template <typename T, int KV>
cudaError_t launch_hd(bool append, const FlPaged& c, void* k, int64_t ks, void* v, int64_t vs, cudaStream_t st)
{
    switch (c.hd) {
    case 64: return launch<T, KV, 64>(append, c, k, ks, v, vs, st);
    case 128: return launch<T, KV, 128>(append, c, k, ks, v, vs, st);
    case 256: return launch<T, KV, 256>(append, c, k, ks, v, vs, st);
    default: return cudaErrorInvalidValue;
    }
}

template <typename T>
cudaError_t launch_kv(bool append, const FlPaged& c, void* k, int64_t ks, void* v, int64_t vs, cudaStream_t st)
{
    switch (c.kv_dtype) {
    case FL_KV_F16: return launch_hd<T, FL_KV_F16>(append, c, k, ks, v, vs, st);
    case FL_KV_Q8: return launch_hd<T, FL_KV_Q8>(append, c, k, ks, v, vs, st);
    case FL_KV_F8: return launch_hd<T, FL_KV_F8>(append, c, k, ks, v, vs, st);
    default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_type(bool append, const FlPaged& c, int type, void* k, int64_t ks, void* v, int64_t vs, cudaStream_t st)
{
    switch (type) {
    case 0: return launch_kv<float>(append, c, k, ks, v, vs, st);
    case 1: return launch_kv<__half>(append, c, k, ks, v, vs, st);
    case 30: return launch_kv<__nv_bfloat16>(append, c, k, ks, v, vs, st);
    default: return cudaErrorInvalidValue;
    }
}

} // namespace

cudaError_t fl_launch_kv_append(const FlPaged& c, int type, const void* k, int64_t k_stride, const void* v,
                                int64_t v_stride, cudaStream_t st)
{
    return launch_type(true, c, type, const_cast<void*>(k), k_stride, const_cast<void*>(v), v_stride, st);
}

cudaError_t fl_launch_kv_gather(const FlPaged& c, int type, void* k, int64_t k_stride, void* v, int64_t v_stride,
                                cudaStream_t st)
{
    return launch_type(false, c, type, k, k_stride, v, v_stride, st);
}
