/*
 * fl_paged_attn.cu — attention of new rows over a paged KV cache
 * (fl_attn_paged_device), the streaming kernel: few query rows against long
 * sequences, bound by reading the cache once.
 *
 * One pass over the keys with a running maximum m, sum l and output o per row:
 *   m' = max(m, x), o = o 2^(m - m') + 2^(x - m') v, l likewise,
 * scores x in units of log2.  Work is cut into items (sequence, kv head, tile
 * of 16 query rows, heads of a group folded into the rows) of 16-key tiles; the
 * tiles of all items, in order, are dealt to the CTAs in equal contiguous
 * ranges, so ragged batches and single long sequences both fill the machine.
 * A range that covers an item whole writes its output; the ranges that share
 * an item leave (o, m, l) in the workspace, merged in range order by a second
 * kernel, so results are the same each time.
 *
 * Each warp takes every fourth 16-key tile of its CTA's range.  Its lanes copy
 * exactly the 16-byte pieces that they later use as matrix fragments into a
 * ring in shared memory (cp.async), so the ring needs no barrier: the copies
 * are the lane's own, and stay in flight while older tiles are computed.
 *
 * S = Q K^T and O += P V run on mma.m16n8k16 (fp16 in, fp32 out): int8 and e4m3
 * elements are exact in fp16, the scale of a key multiplies its score and the
 * scale of a value its weight, in fp32.  The product's inner index may be
 * permuted freely, which is what lets a lane use 16 contiguous bytes of a key
 * as its fragments of four steps, and the score fragments as the weights'
 * operand without a shuffle.
 *  - q is scaled per row by a power of two to a largest magnitude in [2^14,
 *    2^15): 16-bit queries are then exact in fp16 (bf16: down to 2^-38 of the
 *    row's largest), 32-bit ones are two fp16 (22 bits), at twice the products.
 *  - weights p <= 1 carry the value's scale, brought by a power of two to at
 *    most 2^15, so that fp16 keeps 11 bits of every weight down to 2^-29 of the
 *    largest; 32-bit outputs use two fp16 again.  l sums the unrounded weights.
 */
#include "fl_paged.cuh"

namespace {

constexpr int kThreads = 128, kWarps = 4;
constexpr int kRows = 16;     /* query rows of an item */
constexpr int kTile = 16;     /* keys of a tile: never crosses a page */
constexpr int kMinTiles = 8;  /* tiles of a CTA's range, at least: two per warp */
constexpr int kMaxCtas = 148 * 4;

/* ── the schedule ───────────────────────────────────────────────────────── */
struct SeqWork {
    int row0, n, first, len; /* packed rows, their count, the first one's position, keys that are mapped at most */
    int tile0, tiles, items; /* first 16-key tile, tiles of an item (1 when there are no keys), items */
};

__device__ __forceinline__ SeqWork seq_work(const FlPaged& c, int grp, int window, int s)
{
    SeqWork w;
    const int r0 = max(__ldg(c.row_start + s), 0), r1 = min(__ldg(c.row_start + s + 1), c.n_rows);
    const int len = __ldg(c.seq_len + s);
    w.row0 = r0;
    w.n = max(r1 - r0, 0);
    w.first = len - w.n;
    w.len = max(0, min(len, c.cols << c.page_shift));
    const int lo = window > 0 ? max(0, w.first + 1 - window) : 0;
    w.tile0 = lo / kTile;
    w.tiles = max(1, (w.len + kTile - 1) / kTile - w.tile0);
    w.items = w.n > 0 ? c.n_kv * ((w.n * grp + kRows - 1) / kRows) : 0;
    return w;
}

struct Schedule {
    long long total; /* tiles of all items */
    int ctas;        /* ranges */
    __device__ __forceinline__ long long begin(int c) const { return total * c / ctas; }
    __device__ __forceinline__ int owner(long long t) const { return (int)(((t + 1) * ctas - 1) / total); }
};

/* Workspace: Schedule, then the first tile of each sequence, then the
 * partials' (m, l) and outputs, two slots per CTA: [2c] for a range that
 * continues an item, [2c + 1] for one that starts it. */
struct Workspace {
    Schedule* sched;
    long long* seq_tile;
    float2* ml;
    float* o;
};
__host__ __device__ __forceinline__ size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }
__host__ __device__ __forceinline__ Workspace workspace(void* p, int n_seqs, size_t* bytes, int hd)
{
    uint8_t* b = static_cast<uint8_t*>(p);
    Workspace w;
    size_t at = 0;
    w.sched = reinterpret_cast<Schedule*>(b + at);
    at += 256;
    w.seq_tile = reinterpret_cast<long long*>(b + at);
    at += align256((size_t)n_seqs * 8);
    w.ml = reinterpret_cast<float2*>(b + at);
    at += align256((size_t)2 * kMaxCtas * kRows * 8);
    w.o = reinterpret_cast<float*>(b + at);
    at += (size_t)2 * kMaxCtas * kRows * hd * 4;
    if (bytes) *bytes = at;
    return w;
}

/* ── fragments ──────────────────────────────────────────────────────────── */
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ uint32_t pack_half2(float a, float b) { return half2_bits(__floats2half2_rn(a, b)); }

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

/* Bytes 0, 1 (and 2, 3) of w as two halves. */
template <int KV>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi)
{
    if constexpr (KV == FL_KV_Q8) {
        /* 0x6400 + u is the half 1024 + u; u = q + 128 */
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        lo = half2_bits(__hsub2(*reinterpret_cast<const __half2*>(&a), bias));
        hi = half2_bits(__hsub2(*reinterpret_cast<const __half2*>(&b), bias));
    } else {
        const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
        const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
        lo = (uint32_t)a.x | ((uint32_t)a.y << 16);
        hi = (uint32_t)b.x | ((uint32_t)b.y << 16);
    }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int KV, int HD, bool SPLIT>
struct Cfg {
    static constexpr int ES = KV == FL_KV_F16 ? 2 : 1;
    static constexpr int ROW = HD * ES;           /* bytes of a position of one head */
    static constexpr int KC = ROW / 64;           /* 16-byte pieces of a key per lane */
    static constexpr int VB = ROW / 8;            /* bytes of a value per lane */
    static constexpr int VC = VB >= 16 ? VB / 16 : 1;
    static constexpr int VP = VB >= 16 ? 16 : 8;  /* bytes of a value piece */
    static constexpr int KBYTES = kTile * ROW, SCALES = ES == 1 ? 2 * kTile * 4 : 0;
    static constexpr int STAGE = 2 * KBYTES + SCALES;
    static constexpr int STAGES = STAGE <= 4608 ? 4 : STAGE <= 9216 ? 3 : 2;
    static constexpr int NT = HD / 8;             /* 8-wide output tiles */
    static constexpr int KS = HD / 16;            /* inner steps of a score */
    static constexpr int QBYTES = KS * 512 * (SPLIT ? 2 : 1);
    static constexpr int RING = kWarps * STAGES * STAGE;
    static constexpr int MERGE = kWarps * kRows * (HD + 4) * 4;
    static constexpr int SMEM = QBYTES + (RING > MERGE ? RING : MERGE);
    static constexpr bool QREG = KS * (SPLIT ? 8 : 4) <= 32;
    static constexpr int CTAS = HD == 256 ? (SMEM > 113 * 1024 ? 1 : 2) : (SMEM > 75 * 1024 ? 2 : 3);
};

/* First inner element of step k's fragment for lane t: four consecutive ones. */
template <int KV>
__device__ __forceinline__ int q_elem(int k, int t)
{
    return KV == FL_KV_F16 ? (k >> 1) * 32 + t * 8 + (k & 1) * 4 : (k >> 2) * 64 + t * 16 + (k & 3) * 4;
}

template <typename T, int KV, int HD>
__global__ void __launch_bounds__(kThreads, Cfg<KV, HD, sizeof(T) == 4>::CTAS)
    paged_stream_kernel(const FlPaged c, const FlPagedAttn a)
{
    constexpr bool SPLIT = sizeof(T) == 4;
    using C = Cfg<KV, HD, SPLIT>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long s_scan[kWarps];
    __shared__ long long s_at;
    __shared__ int s_seq;
    __shared__ float s_fr[kRows];                  /* score units of a row's scaled q */
    __shared__ float2 s_ml[kWarps][kRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int grp = a.n_heads / c.n_kv;
    Workspace ws = workspace(a.workspace, c.n_seqs, nullptr, HD);

    /* ── this CTA's range: a scan over the sequences' tiles ── */
    const int per = (c.n_seqs + kThreads - 1) / kThreads;
    long long mine = 0;
    for (int s = tid * per; s < min(c.n_seqs, (tid + 1) * per); s++) {
        const SeqWork w = seq_work(c, grp, a.window, s);
        mine += (long long)w.items * w.tiles;
    }
    long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += u;
    }
    if (lane == 31) s_scan[warp] = before;
    if (tid == 0) s_seq = -1;
    __syncthreads();
    Schedule sc;
    sc.total = 0;
    before -= mine;
    for (int w = 0; w < kWarps; w++) {
        if (w < warp) before += s_scan[w];
        sc.total += s_scan[w];
    }
    sc.ctas = (int)min((long long)gridDim.x, max(1ll, sc.total / kMinTiles));
    const bool in = sc.total > 0 && (int)blockIdx.x < sc.ctas;
    const long long w0 = in ? sc.begin(blockIdx.x) : 0, w1 = in ? sc.begin(blockIdx.x + 1) : 0;
    if (blockIdx.x == 0) {
        if (tid == 0) *ws.sched = sc;
    }
    {
        long long at = before;
        const bool find = w0 < w1 && before <= w0 && w0 < before + mine;
        if (find || blockIdx.x == 0) {
            for (int s = tid * per; s < min(c.n_seqs, (tid + 1) * per); s++) {
                const SeqWork w = seq_work(c, grp, a.window, s);
                const long long n = (long long)w.items * w.tiles;
                if (blockIdx.x == 0) ws.seq_tile[s] = at;
                if (find && at <= w0 && w0 < at + n) s_seq = s, s_at = at;
                at += n;
            }
        }
    }
    __syncthreads();
    int seq = s_seq;
    long long seq_at = s_at;
    if (seq < 0) return;

    const uint32_t q_smem = fl_smem_u32(smem);
    const uint32_t ring = q_smem + C::QBYTES + warp * (C::STAGES * C::STAGE);
    const uint4* q_frag = reinterpret_cast<const uint4*>(smem);
    float* merge = reinterpret_cast<float*>(smem + C::QBYTES);
    SeqWork sw = seq_work(c, grp, a.window, seq);

    for (long long at = w0; at < w1;) {
        while (at >= seq_at + (long long)sw.items * sw.tiles) {
            seq_at += (long long)sw.items * sw.tiles;
            sw = seq_work(c, grp, a.window, ++seq);
        }
        /* the segment: tiles [j0, j1) of item (head, row tile) */
        const int item = (int)((at - seq_at) / sw.tiles);
        const long long item_at = seq_at + (long long)item * sw.tiles;
        const int j0 = (int)(at - item_at), j1 = (int)min((long long)sw.tiles, w1 - item_at);
        const int nrt = sw.items / c.n_kv, head = item / nrt, rt = item - head * nrt;
        const int R = sw.n * grp;
        at = item_at + j1;

        /* ── q fragments ── */
        for (int r = warp; r < kRows; r += kWarps) {
            const int f = rt * kRows + r, i = f / grp;
            const T* q = static_cast<const T*>(a.q) + (int64_t)(sw.row0 + i) * a.q_stride +
                         (int64_t)(head * grp + f - i * grp) * HD;
            float x[HD / 32];
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < HD / 32; e++) {
                x[e] = f < R ? fl_to_float(q[lane + 32 * e]) : 0.0f;
                top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            /* q 2^up has its largest magnitude in [2^14, 2^15) */
            int up = 0;
            if (top != 0 && top < 0x7f800000u) up = 14 - ilogbf(__uint_as_float(top));
            if (lane == 0) s_fr[r] = ldexpf(a.softcap > 0.0f ? a.scale / a.softcap : a.scale * 1.44269504f, -up);
            /* into fragment order: row r of step k, lane (r % 8) * 4 + t, element pairs at words r / 8 and r / 8 + 2 */
#pragma unroll
            for (int e = 0; e < HD / 32; e++) {
                const int d = lane + 32 * e;
                const float y = ldexpf(x[e], up);
                const __half hi = __float2half_rn(y);
                int k, tt, i4;
                if (KV == FL_KV_F16) {
                    k = (d >> 5) * 2 + ((d >> 2) & 1), tt = (d >> 3) & 3, i4 = d & 3;
                } else {
                    k = (d >> 6) * 4 + ((d >> 2) & 3), tt = (d >> 4) & 3, i4 = d & 3;
                }
                __half* dst = reinterpret_cast<__half*>(smem) + (k * 32 + (r & 7) * 4 + tt) * 8 + (r >> 3) * 2 +
                              (i4 >> 1) * 4 + (i4 & 1);
                dst[0] = hi;
                if (SPLIT) dst[C::KS * 256] = __float2half_rn(y - __half2float(hi));
            }
        }
        __syncthreads();
        uint4 qf[C::QREG ? C::KS : 1], ql[C::QREG && SPLIT ? C::KS : 1];
        if constexpr (C::QREG) {
#pragma unroll
            for (int k = 0; k < C::KS; k++) {
                qf[k] = q_frag[k * 32 + lane];
                if (SPLIT) ql[k] = q_frag[(C::KS + k) * 32 + lane];
            }
        }
        const float fr[2] = {s_fr[g], s_fr[g + 8]};
        int pos[2]; /* last key of rows g, g + 8; rows past R see nothing */
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int f = rt * kRows + g + 8 * i;
            pos[i] = f < R ? sw.first + f / grp : -1;
        }
        /* of the item's rows: the first and the last position */
        const int pos_min = sw.first + rt * kRows / grp, pos_max = sw.first + min(R - 1, rt * kRows + kRows - 1) / grp;
        const int win = a.window > 0 ? a.window : INT_MAX;

        /* ── the warp's tiles: j0 + warp, + 4, ... ── */
        const int n_mine = j1 - j0 > warp ? (j1 - j0 - warp + kWarps - 1) / kWarps : 0;
        const int32_t* table = c.table + (size_t)seq * c.cols;
        int pages = -1; /* lane i: the page of the warp's tile (i0 & ~31) + i */
        auto load_pages = [&](int i0) {
            const int i = i0 + lane;
            pages = -1;
            if (i < n_mine) {
                const int key = (sw.tile0 + j0 + warp + i * kWarps) * kTile;
                if (key < sw.len) pages = __ldg(table + (key >> c.page_shift));
                if ((unsigned)pages >= (unsigned)c.n_pages) pages = -1;
            }
        };
        int held = -1; /* the tile block whose pages are held */
        auto fetch = [&](int i) { /* copies of tile i into stage i % STAGES; true when it is mapped */
            if (i < n_mine) {
                if ((i >> 5) != held) {
                    held = i >> 5;
                    load_pages(held << 5);
                }
                const int page = __shfl_sync(0xffffffffu, pages, i & 31);
                if (page >= 0) {
                    const int key = (sw.tile0 + j0 + warp + i * kWarps) * kTile;
                    const int64_t row = (((int64_t)page * c.n_kv + head) << c.page_shift) + (key & ((1 << c.page_shift) - 1));
                    const uint32_t dst = ring + (i % C::STAGES) * C::STAGE;
                    const uint8_t* kp = static_cast<const uint8_t*>(c.k) + row * C::ROW + ((g >> 1) * 4 + (g & 1)) * C::ROW + t * 16;
                    const uint8_t* vp = static_cast<const uint8_t*>(c.v) + row * C::ROW + t * 4 * C::ROW + g * C::VP;
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int p = 0; p < C::KC; p++)
                            cp_async16(dst + (n * C::KC + p) * 512 + lane * 16, kp + n * 2 * C::ROW + p * 64);
#pragma unroll
                    for (int n = 0; n < 4; n++)
#pragma unroll
                        for (int p = 0; p < C::VC; p++) {
                            const uint32_t d = dst + C::KBYTES + (n * C::VC + p) * (32 * C::VP) + lane * C::VP;
                            if (C::VP == 16)
                                cp_async16(d, vp + n * C::ROW + p * 128);
                            else
                                cp_async8(d, vp + n * C::ROW);
                        }
                    if (C::SCALES && lane < 8)
                        cp_async16(dst + 2 * C::KBYTES + lane * 16, (lane < 4 ? c.k_scale : c.v_scale) + row + (lane & 3) * 4);
                }
            }
            cp_async_commit();
        };

        float acc[C::NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        int ev = -1000; /* exponent of the values' scales that acc counts in (8 bits) */
#pragma unroll
        for (int n = 0; n < C::NT; n++) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;

#pragma unroll
        for (int i = 0; i < C::STAGES - 1; i++) fetch(i);
        int cur_held = -1, cur_pages = -1;
        for (int i = 0; i < n_mine; i++) {
            if ((i >> 5) != cur_held) { /* the pages of the tiles being computed lag those being fetched */
                cur_held = i >> 5;
                const int keep = pages;
                load_pages(cur_held << 5);
                cur_pages = pages;
                pages = keep;
            }
            fetch(i + C::STAGES - 1);
            if (__shfl_sync(0xffffffffu, cur_pages, i & 31) < 0) continue;
            cp_async_wait<C::STAGES - 1>();
            __syncwarp(); /* the scales are other lanes' copies */
            const uint8_t* st = smem + C::QBYTES + warp * (C::STAGES * C::STAGE) + (i % C::STAGES) * C::STAGE;
            const int key0 = (sw.tile0 + j0 + warp + i * kWarps) * kTile;

            /* scores: s[n][..] of keys 4t + 2n + {0, 1}, rows g and g + 8 */
            float s[2][4] = {};
#pragma unroll
            for (int p = 0; p < C::KC; p++) {
                const uint4 k0 = *reinterpret_cast<const uint4*>(st + p * 512 + lane * 16);
                const uint4 k1 = *reinterpret_cast<const uint4*>(st + (C::KC + p) * 512 + lane * 16);
                const uint32_t w0_[4] = {k0.x, k0.y, k0.z, k0.w}, w1_[4] = {k1.x, k1.y, k1.z, k1.w};
                constexpr int STEPS = KV == FL_KV_F16 ? 2 : 4;
#pragma unroll
                for (int e = 0; e < STEPS; e++) {
                    const int k = p * STEPS + e;
                    uint32_t b[2][2];
                    if constexpr (KV == FL_KV_F16) {
                        b[0][0] = w0_[2 * e], b[0][1] = w0_[2 * e + 1];
                        b[1][0] = w1_[2 * e], b[1][1] = w1_[2 * e + 1];
                    } else {
                        widen<KV>(w0_[e], b[0][0], b[0][1]);
                        widen<KV>(w1_[e], b[1][0], b[1][1]);
                    }
                    if (SPLIT) {
                        const uint4 lo = C::QREG ? ql[C::QREG ? k : 0] : q_frag[(C::KS + k) * 32 + lane];
                        mma_f16(s[0], lo, b[0][0], b[0][1]);
                        mma_f16(s[1], lo, b[1][0], b[1][1]);
                    }
                    const uint4 hi = C::QREG ? qf[C::QREG ? k : 0] : q_frag[k * 32 + lane];
                    mma_f16(s[0], hi, b[0][0], b[0][1]);
                    mma_f16(s[1], hi, b[1][0], b[1][1]);
                }
            }
            float sv[4];
            if constexpr (C::SCALES != 0) {
                const float4 k4 = reinterpret_cast<const float4*>(st + 2 * C::KBYTES)[t];
                const float4 v4 = reinterpret_cast<const float4*>(st + 2 * C::KBYTES + 64)[t];
                s[0][0] *= k4.x, s[0][2] *= k4.x, s[0][1] *= k4.y, s[0][3] *= k4.y;
                s[1][0] *= k4.z, s[1][2] *= k4.z, s[1][1] *= k4.w, s[1][3] *= k4.w;
                sv[0] = v4.x, sv[1] = v4.y, sv[2] = v4.z, sv[3] = v4.w;
            }
            /* keys that no row, or only some rows, may see */
            const bool masked = key0 + kTile - 1 > pos_min || key0 + kTile > sw.len || pos_max - key0 >= win;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float x = s[n][e] * fr[e >> 1];
                    if (a.softcap > 0.0f) x = tanhf(x) * (a.softcap * 1.44269504f);
                    if (masked) {
                        const int key = key0 + 4 * t + 2 * n + (e & 1);
                        const bool see = key <= pos[e >> 1] && pos[e >> 1] - key < win && key < sw.len;
                        x = see ? x : -INFINITY;
                    }
                    s[n][e] = x;
                }
            if (masked && C::SCALES) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int key = key0 + 4 * t + e;
                    if (key > pos_max || key >= sw.len || pos_min - key >= win) sv[e] = 0.0f;
                }
            }
            /* running maximum; the exponent of the values' scales likewise */
            float alpha[2];
            bool moved = false;
#pragma unroll
            for (int i2 = 0; i2 < 2; i2++) {
                float mx = fmaxf(fmaxf(s[0][2 * i2], s[0][2 * i2 + 1]), fmaxf(s[1][2 * i2], s[1][2 * i2 + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[i2], mx);
                alpha[i2] = 1.0f;
                if (mn > m[i2]) {
                    alpha[i2] = ex2(m[i2] - mn); /* 0 the first time */
                    m[i2] = mn;
                    moved = true;
                }
            }
            float up = 16384.0f, down = 1.0f; /* 2^14; what a larger exponent makes of acc */
            if constexpr (C::SCALES != 0) {
                /* the exponent bits of the largest finite scale */
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t b = __float_as_uint(sv[e]) & 0x7fffffffu;
                    if (b < 0x7f800000u) top = max(top, b);
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int en = max((int)(top >> 23) - 127, -100);
                if (en > ev) {
                    down = ev == -1000 ? 0.0f : ex2((float)(ev - en));
                    ev = en;
                    moved = true;
                }
                up = __int_as_float((127 + 14 - ev) << 23);
            }
            if (__any_sync(0xffffffffu, moved)) {
                l[0] *= alpha[0];
                l[1] *= alpha[1];
                alpha[0] *= down;
                alpha[1] *= down;
#pragma unroll
                for (int n = 0; n < C::NT; n++) {
                    acc[n][0] *= alpha[0], acc[n][1] *= alpha[0];
                    acc[n][2] *= alpha[1], acc[n][3] *= alpha[1];
                }
            }
            /* weights, in the layout of the first operand */
            float p[2][4];
#pragma unroll
            for (int i2 = 0; i2 < 2; i2++) {
                const float ref = m[i2] == -INFINITY ? 0.0f : m[i2];
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float w = ex2(s[n][2 * i2 + e] - ref);
                        l[i2] += w;
                        if (C::SCALES) {
                            w *= sv[2 * n + e] * up;
                            if (masked && s[n][2 * i2 + e] == -INFINITY) w = 0.0f;
                        } else {
                            w *= up;
                        }
                        p[n][2 * i2 + e] = w;
                    }
            }
            uint4 pa, pl;
            pa.x = pack_half2(p[0][0], p[0][1]);
            pa.y = pack_half2(p[0][2], p[0][3]);
            pa.z = pack_half2(p[1][0], p[1][1]);
            pa.w = pack_half2(p[1][2], p[1][3]);
            if (SPLIT) {
                auto rest = [](uint32_t h, float x0, float x1) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                    return pack_half2(x0 - f.x, x1 - f.y);
                };
                pl.x = rest(pa.x, p[0][0], p[0][1]);
                pl.y = rest(pa.y, p[0][2], p[0][3]);
                pl.z = rest(pa.z, p[1][0], p[1][1]);
                pl.w = rest(pa.w, p[1][2], p[1][3]);
            }
            /* values: keys 4t..4t+3 at the lane's elements; tile n of the output holds element n of every lane's run */
            uint4 seen; /* masked tiles of types that hold NaN or infinity: 1 where a row sees a key */
            if (masked && KV != FL_KV_Q8) {
                auto one = [&](int n, int i2) {
                    return (s[n][2 * i2] > -INFINITY || s[n][2 * i2] != s[n][2 * i2] ? 0x3c00u : 0u) |
                           (s[n][2 * i2 + 1] > -INFINITY || s[n][2 * i2 + 1] != s[n][2 * i2 + 1] ? 0x3c000000u : 0u);
                };
                seen = make_uint4(one(0, 0), one(0, 1), one(1, 0), one(1, 1));
            }
#pragma unroll
            for (int pc = 0; pc < C::VC; pc++) {
                uint32_t w[4][4];
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const uint8_t* src = st + C::KBYTES + (n * C::VC + pc) * (32 * C::VP) + lane * C::VP;
                    if (C::VP == 16) {
                        const uint4 u = *reinterpret_cast<const uint4*>(src);
                        w[n][0] = u.x, w[n][1] = u.y, w[n][2] = u.z, w[n][3] = u.w;
                    } else {
                        const uint2 u = *reinterpret_cast<const uint2*>(src);
                        w[n][0] = u.x, w[n][1] = u.y;
                    }
                }
                constexpr int PER = KV == FL_KV_F16 ? 2 : 4; /* elements of a word */
#pragma unroll
                for (int x = 0; x < C::VP / 4; x++) {
                    uint32_t b0[PER], b1[PER];
                    if constexpr (KV == FL_KV_F16) {
                        b0[0] = __byte_perm(w[0][x], w[1][x], 0x5410), b0[1] = __byte_perm(w[0][x], w[1][x], 0x7632);
                        b1[0] = __byte_perm(w[2][x], w[3][x], 0x5410), b1[1] = __byte_perm(w[2][x], w[3][x], 0x7632);
                    } else {
                        widen<KV>(__byte_perm(w[0][x], w[1][x], 0x5140), b0[0], b0[1]);
                        widen<KV>(__byte_perm(w[0][x], w[1][x], 0x7362), b0[2], b0[3]);
                        widen<KV>(__byte_perm(w[2][x], w[3][x], 0x5140), b1[0], b1[1]);
                        widen<KV>(__byte_perm(w[2][x], w[3][x], 0x7362), b1[2], b1[3]);
                    }
#pragma unroll
                    for (int e = 0; e < PER; e++) {
                        const int n = pc * (C::VP / C::ES) + x * PER + e;
                        if (KV != FL_KV_Q8 && masked) {
                            /* a weight of 0 does not keep NaN or infinity out of a sum: where the tile holds one, it
                             * is left out, and made NaN in the rows that see it */
                            auto odd = [](uint32_t h) { return (h & 0x7c00u) == 0x7c00u || (h & 0x7c000000u) == 0x7c000000u; };
                            if (__any_sync(0xffffffffu, odd(b0[e]) || odd(b1[e]))) {
                                auto flag = [](uint32_t h) {
                                    return ((h & 0x7c00u) == 0x7c00u ? 0x3c00u : 0u) |
                                           ((h & 0x7c000000u) == 0x7c000000u ? 0x3c000000u : 0u);
                                };
                                const uint32_t f0 = flag(b0[e]), f1 = flag(b1[e]);
                                float hit[4] = {};
                                mma_f16(hit, seen, f0, f1);
#pragma unroll
                                for (int z = 0; z < 4; z++)
                                    if (hit[z] > 0.0f) acc[n][z] = __uint_as_float(0x7fffffffu);
                                b0[e] &= ~((f0 & 0x3c00u ? 0xffffu : 0u) | (f0 & 0x3c000000u ? 0xffff0000u : 0u));
                                b1[e] &= ~((f1 & 0x3c00u ? 0xffffu : 0u) | (f1 & 0x3c000000u ? 0xffff0000u : 0u));
                            }
                        }
                        if (SPLIT) mma_f16(acc[n], pl, b0[e], b1[e]);
                        mma_f16(acc[n], pa, b0[e], b1[e]);
                    }
                }
            }
            __syncwarp(); /* the stage's scales are read before another lane's copy may land there */
        }
        cp_async_wait<0>();

        /* ── the CTA's warps, merged in order ── */
#pragma unroll
        for (int i = 0; i < 2; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (t == 0) s_ml[warp][g + 8 * i] = make_float2(m[i], l[i]);
        }
        __syncthreads(); /* every warp is done with its ring, too */
        const float unit = C::SCALES ? ldexpf(1.0f, (ev == -1000 ? 0 : ev) - 14) : 6.1035156e-05f; /* 2^-14 */
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = g + 8 * i;
            float M = -INFINITY;
            for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_ml[w][r].x);
            const float f = m[i] == -INFINITY ? 0.0f : ex2(m[i] - M) * unit;
            float* dst = merge + (warp * kRows + r) * (HD + 4);
#pragma unroll
            for (int n = 0; n < C::NT; n++) {
                constexpr int RUN = C::VP / C::ES; /* consecutive elements of a lane */
                const int pc = n / RUN, x = n % RUN;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float v = acc[n][2 * i + e];
                    dst[pc * 8 * RUN + (2 * t + e) * RUN + x] = m[i] == -INFINITY ? 0.0f : v * f;
                }
            }
        }
        __syncthreads();
        const bool whole = j0 == 0 && j1 == sw.tiles;
        const int slot = 2 * (int)blockIdx.x + (j0 == 0 ? 1 : 0);
        for (int x = tid; x < kRows * HD / 8; x += kThreads) {
            const int r = x / (HD / 8), d = (x - r * (HD / 8)) * 8, f = rt * kRows + r;
            if (f >= R) break;
            float o[8] = {}, M = -INFINITY, L = 0.0f;
            for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_ml[w][r].x);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float2 ml = s_ml[w][r];
                L += ml.x == -INFINITY ? ml.y : ml.y * ex2(ml.x - M);
                const float4* src = reinterpret_cast<const float4*>(merge + (w * kRows + r) * (HD + 4) + d);
                const float4 u = src[0], v = src[1];
                o[0] += u.x, o[1] += u.y, o[2] += u.z, o[3] += u.w, o[4] += v.x, o[5] += v.y, o[6] += v.z, o[7] += v.w;
            }
            if (whole) {
                const int i = f / grp, h = head * grp + f - i * grp;
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
                for (int e = 0; e < 8; e++) o[e] *= inv;
                fl_store8(static_cast<T*>(a.out) + (int64_t)(sw.row0 + i) * a.out_stride + (int64_t)h * HD + d, o);
                if (a.lse && d == 0)
                    a.lse[(int64_t)(sw.row0 + i) * a.n_heads + h] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.693147181f;
            } else {
                fl_store8(ws.o + ((size_t)slot * kRows + r) * HD + d, o);
                if (d == 0) ws.ml[slot * kRows + r] = make_float2(M, L);
            }
        }
        __syncthreads(); /* merge and q are free again */
    }
}

/* Items that several ranges share: the partials in range order. */
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) paged_merge_kernel(const FlPaged c, const FlPagedAttn a)
{
    constexpr int LANES = HD / 8, PER_WARP = 32 / LANES; /* lanes of a (row, head), their number in a warp */
    const int lane = threadIdx.x & 31;
    fl_pdl_wait();
    const Workspace ws = workspace(a.workspace, c.n_seqs, nullptr, HD);
    const int64_t n_pairs = (int64_t)c.n_rows * a.n_heads;
    const int64_t pair0 = (((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5) * PER_WARP;
    if (pair0 >= n_pairs) return;
    const int64_t pair = pair0 + lane / LANES;
    const int d = (lane % LANES) * 8;
    const int grp = a.n_heads / c.n_kv;
    int prev = -1, at_seq = -1, seq = -1;
#pragma unroll
    for (int i = 0; i < PER_WARP; i++) {
        if (pair0 + i >= n_pairs) break;
        const int row = (int)((pair0 + i) / a.n_heads);
        if (row != prev) at_seq = fl_row_seq(c.row_start, c.n_seqs, row);
        prev = row;
        if (i == lane / LANES) seq = at_seq;
    }
    if (seq < 0) return;
    const int row = (int)(pair / a.n_heads), h = (int)(pair - (int64_t)row * a.n_heads);
    const SeqWork sw = seq_work(c, grp, a.window, seq);
    const Schedule sc = *ws.sched;
    const int head = h / grp, f = (row - sw.row0) * grp + h - head * grp;
    const int nrt = sw.items / c.n_kv, item = head * nrt + f / kRows, r = f % kRows;
    const long long t0 = ws.seq_tile[seq] + (long long)item * sw.tiles;
    const int c0 = sc.owner(t0), c1 = sc.owner(t0 + sw.tiles - 1);
    if (c0 == c1) return; /* written by its range */
    float M = -INFINITY;
    for (int i = c0; i <= c1; i++) M = fmaxf(M, ws.ml[(2 * i + (i == c0)) * kRows + r].x);
    float o[8] = {}, L = 0.0f;
    for (int i = c0; i <= c1; i++) {
        const int at = (2 * i + (i == c0)) * kRows + r;
        const float2 ml = ws.ml[at];
        const float w = ml.x == -INFINITY ? 0.0f : ex2(ml.x - M);
        L += ml.x == -INFINITY ? ml.y : ml.y * w;
        const float4* src = reinterpret_cast<const float4*>(ws.o + (size_t)at * HD + d);
        const float4 u = src[0], v = src[1];
        const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = fmaf(x[e], w, o[e]);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] *= inv;
    fl_store8(static_cast<T*>(a.out) + (int64_t)row * a.out_stride + (int64_t)h * HD + d, o);
    if (a.lse && d == 0) a.lse[pair] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.693147181f;
}

template <typename T, int KV, int HD>
cudaError_t launch(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    using C = Cfg<KV, HD, sizeof(T) == 4>;
    static_assert(C::CTAS * 148 <= kMaxCtas, "workspace slots");
    static int sms[64] = {}; /* SMs of a device, once its kernel is configured */
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!sms[dev]) {
        e = cudaFuncSetAttribute(paged_stream_kernel<T, KV, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        int n = 0;
        e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
        sms[dev] = n < 148 ? n : 148;
    }
    paged_stream_kernel<T, KV, HD><<<sms[dev] * C::CTAS, kThreads, C::SMEM, st>>>(c, a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int64_t pairs = (int64_t)c.n_rows * a.n_heads, per_block = kWarps * (256 / HD);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((pairs + per_block - 1) / per_block));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_merge_kernel<T, HD>, c, a);
}

template <typename T, int KV>
cudaError_t launch_hd(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    switch (c.hd) {
    case 64: return launch<T, KV, 64>(c, a, st);
    case 128: return launch<T, KV, 128>(c, a, st);
    case 256: return launch<T, KV, 256>(c, a, st);
    default: return cudaErrorInvalidValue;
    }
}

template <typename T>
cudaError_t launch_kv(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    switch (c.kv_dtype) {
    case FL_KV_F16: return launch_hd<T, FL_KV_F16>(c, a, st);
    case FL_KV_Q8: return launch_hd<T, FL_KV_Q8>(c, a, st);
    case FL_KV_F8: return launch_hd<T, FL_KV_F8>(c, a, st);
    default: return cudaErrorInvalidValue;
    }
}

} // namespace

size_t fl_paged_attn_workspace(const FlPaged& c, int)
{
    size_t bytes;
    workspace(nullptr, c.n_seqs, &bytes, c.hd);
    return bytes;
}

cudaError_t fl_launch_paged_attn(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    switch (a.type) {
    case 0: return launch_kv<float>(c, a, st);
    case 1: return launch_kv<__half>(c, a, st);
    case 30: return launch_kv<__nv_bfloat16>(c, a, st);
    default: return cudaErrorInvalidValue;
    }
}
