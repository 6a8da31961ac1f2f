/*
 * fl_paged_attn.cu — attention of new rows over a paged KV cache
 * (fl_attn_paged_device).
 *
 * One warp per (row, query head): the lanes hold the head's elements, keys
 * are taken one after another with a running maximum and sum.
 */
#include "fl_paged.cuh"

namespace {

constexpr int kThreads = 128;

template <int KV>
__device__ __forceinline__ float kv_elem(const void* base, int64_t i)
{
    if constexpr (KV == FL_KV_F16) return __half2float(static_cast<const __half*>(base)[i]);
    if constexpr (KV == FL_KV_Q8) return (float)static_cast<const int8_t*>(base)[i];
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const __nv_fp8_storage_t*>(base)[i], __NV_E4M3)));
}

template <typename T, int KV, int HD>
__global__ void __launch_bounds__(kThreads) paged_attn_kernel(const FlPaged c, const FlPagedAttn a)
{
    constexpr int PER = HD / 32;
    const int lane = threadIdx.x & 31;
    const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
    if (item >= (int64_t)c.n_rows * a.n_heads) return;
    const int row = (int)(item / a.n_heads), h = (int)(item - (int64_t)row * a.n_heads);
    const int s = fl_row_seq(c.row_start, c.n_seqs, row);
    if (s < 0) return;
    const int pos = c.seq_len[s] - (c.row_start[s + 1] - row);
    const int kvh = h / (a.n_heads / c.n_kv);
    const T* q = static_cast<const T*>(a.q) + row * a.q_stride + (int64_t)h * HD;
    float qr[PER], o[PER] = {};
#pragma unroll
    for (int i = 0; i < PER; i++) qr[i] = fl_to_float(q[lane + 32 * i]);
    float m = -INFINITY, l = 0.0f;
    const int hi = (int)min((int64_t)pos + 1, (int64_t)c.cols << c.page_shift);
    const int lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    for (int j = lo; j < hi; j++) {
        const int64_t at = fl_cache_row(c, s, j, kvh);
        if (at < 0) continue;
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) x = fmaf(qr[i], kv_elem<KV>(c.k, at * HD + lane + 32 * i), x);
        x = fl_warp_sum(x);
        if (KV != FL_KV_F16) x *= c.k_scale[at];
        x *= a.scale;
        if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
        const float mn = fmaxf(m, x);
        const float corr = mn == -INFINITY ? 1.0f : expf(m - mn);
        const float p = mn == -INFINITY ? 0.0f : expf(x - mn);
        m = mn;
        l = l * corr + p;
        const float pv = KV == FL_KV_F16 ? p : p * c.v_scale[at];
#pragma unroll
        for (int i = 0; i < PER; i++) o[i] = fmaf(pv, kv_elem<KV>(c.v, at * HD + lane + 32 * i), o[i] * corr);
    }
    T* out = static_cast<T*>(a.out) + row * a.out_stride + (int64_t)h * HD;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < PER; i++) out[lane + 32 * i] = fl_from_float<T>(l == 0.0f ? 0.0f : o[i] * inv);
    if (a.lse && lane == 0) a.lse[item] = l == 0.0f ? -INFINITY : m + logf(l);
}

template <typename T, int KV>
cudaError_t launch(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    const int64_t items = (int64_t)c.n_rows * a.n_heads;
    const unsigned grid = (unsigned)((items + 3) / 4);
    switch (c.hd) {
    case 64: paged_attn_kernel<T, KV, 64><<<grid, kThreads, 0, st>>>(c, a); break;
    case 128: paged_attn_kernel<T, KV, 128><<<grid, kThreads, 0, st>>>(c, a); break;
    case 256: paged_attn_kernel<T, KV, 256><<<grid, kThreads, 0, st>>>(c, a); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_kv(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    switch (c.kv_dtype) {
    case FL_KV_F16: return launch<T, FL_KV_F16>(c, a, st);
    case FL_KV_Q8: return launch<T, FL_KV_Q8>(c, a, st);
    case FL_KV_F8: return launch<T, FL_KV_F8>(c, a, st);
    default: return cudaErrorInvalidValue;
    }
}

} // namespace

size_t fl_paged_attn_workspace(const FlPaged&, int) { return 256; }

cudaError_t fl_launch_paged_attn(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    switch (a.type) {
    case 0: return launch_kv<float>(c, a, st);
    case 1: return launch_kv<__half>(c, a, st);
    case 30: return launch_kv<__nv_bfloat16>(c, a, st);
    default: return cudaErrorInvalidValue;
    }
}
