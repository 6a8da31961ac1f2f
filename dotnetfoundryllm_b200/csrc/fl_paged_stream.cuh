/*
 * fl_paged_stream.cuh — attention of new rows over a paged KV cache
 * (fl_attn_paged_device), the streaming kernel: few query rows against long
 * sequences, bound by reading the cache once.  Included by one source file
 * per head dimension.
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
#ifndef FL_PAGED_STREAM_CUH
#define FL_PAGED_STREAM_CUH

#include <atomic>
#include <climits>

#include "fl_paged.cuh"

namespace flps {
namespace {

constexpr int kThreads = 128, kWarps = 4;
constexpr int kRows = 16;     /* query rows of an item */
constexpr int kTile = 16;     /* keys of a tile: never crosses a page */
constexpr int kItemCost = 24; /* what starting an item costs, in tiles */
constexpr int kMinUnits = 8;  /* a range is at least this long: two tiles per warp */
constexpr int kMaxCtas = 148 * 4;

/* ── the schedule ───────────────────────────────────────────────────────── */
struct SeqWork {
    int row0, n, first, len; /* packed rows, their count, the first one's position, keys that are mapped at most */
    int tile0, tiles, nrt;   /* first 16-key tile, tiles of an item (1 when there are no keys), row tiles */
    uint32_t cost, units;    /* of an item, of the sequence: kItemCost + tiles, the tiles the last of them */
};

__device__ __forceinline__ SeqWork seq_work(const FlPaged& c, const FlPagedAttn& a, int s)
{
    SeqWork w;
    const int r0 = max(__ldg(c.row_start + s), 0), r1 = min(__ldg(c.row_start + s + 1), c.n_rows);
    const int len = fl_seq_len(c, s);
    w.row0 = r0;
    w.n = max(r1 - r0, 0);
    w.first = len - w.n;
    w.len = min(len, c.cols << c.page_shift);
    w.tile0 = fl_first_seen(w.first, a.window) / kTile;
    w.tiles = max(1, (w.len + kTile - 1) / kTile - w.tile0);
    w.nrt = (w.n * a.grp + kRows - 1) / kRows;
    w.cost = kItemCost + w.tiles;
    w.units = (uint32_t)(c.n_kv * w.nrt) * w.cost;
    return w;
}

/* ── fragments ──────────────────────────────────────────────────────────── */
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

/* d += (lo + hi) b with the sum over steps rounded to nearest: the tensor core truncates its sums, which over a
 * long row of keys adds up to more than fp32 sums would lose. */
__device__ __forceinline__ void mma_f16_add(float (&d)[4], const uint4& lo, const uint4& hi, uint32_t b0, uint32_t b1)
{
    float x[4] = {};
    mma_f16(x, lo, b0, b1);
    mma_f16(x, hi, b0, b1);
#pragma unroll
    for (int i = 0; i < 4; i++) d[i] += x[i];
}

/* All bits of the halves of h that are NaN or infinite. */
__device__ __forceinline__ uint32_t odd_halves(uint32_t h)
{
    return ((h & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((h & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
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
    static constexpr int TILE = 2 * KBYTES + SCALES;
    /* tiles a warp takes at once: two where they are small, for shorter chains and half the reductions per key */
    static constexpr int U = KBYTES <= 2048 ? 2 : 1;
    static constexpr int STAGE = U * TILE;
    static constexpr int STAGES = STAGE <= 4608 ? 3 : STAGE <= 9216 ? (U == 2 ? 2 : 3) : 2;
    static constexpr int NT = HD / 8;             /* 8-wide output tiles */
    static constexpr int KS = HD / 16;            /* inner steps of a score */
    static constexpr int QBYTES = KS * 512 * (SPLIT ? 2 : 1);
    static constexpr int RING = kWarps * STAGES * STAGE;
    static constexpr int MERGE = kWarps * kRows * (HD + 4) * 4;
    static constexpr int SMEM = QBYTES + (RING > MERGE ? RING : MERGE);
    static constexpr bool QREG = KS * (SPLIT ? 8 : 4) <= 32;
    static constexpr int CTAS = HD == 256 ? (SMEM > 113 * 1024 ? 1 : 2) : (SMEM > 75 * 1024 ? 2 : 3);
};

template <typename T, int KV, int HD>
__global__ void __launch_bounds__(kThreads, Cfg<KV, HD, sizeof(T) == 4>::CTAS)
    paged_stream_kernel(const FlPaged c, const FlPagedAttn a)
{
    constexpr bool SPLIT = sizeof(T) == 4;
    using C = Cfg<KV, HD, SPLIT>;
    constexpr int U = C::U;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t s_scan[kWarps];
    __shared__ uint32_t s_at;
    __shared__ int s_seq;
    __shared__ float s_fr[kRows];                  /* score units of a row's scaled q */
    __shared__ float2 s_ml[kWarps][kRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const FlAttnSpace ws = fl_attn_space(a.workspace, c.n_seqs, kMaxCtas, kRows, HD);
    fl_pdl_trigger(); /* the merge kernel may take its place; it waits for this grid's end */

    /* ── this CTA's range: a scan over the sequences' units ── */
    const int per_thread = (c.n_seqs + kThreads - 1) / kThreads;
    const int s_lo = min(tid * per_thread, c.n_seqs), s_hi = min(s_lo + per_thread, c.n_seqs);
    uint32_t mine = 0;
    for (int s = s_lo; s < s_hi; s++) mine += seq_work(c, a, s).units;
    uint32_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += u;
    }
    if (lane == 31) s_scan[warp] = before;
    if (tid == 0) s_seq = -1;
    __syncthreads();
    struct {
        uint32_t total, per;
    } sc;
    sc.total = 0;
    before -= mine;
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
        if (w < warp) before += s_scan[w];
        sc.total += s_scan[w];
    }
    sc.per = max((uint32_t)kMinUnits, (sc.total + gridDim.x - 1) / gridDim.x);
    const unsigned long long w0_64 = (unsigned long long)blockIdx.x * sc.per;
    const uint32_t w0 = (uint32_t)min(w0_64, (unsigned long long)sc.total);
    const uint32_t w1 = (uint32_t)min(w0_64 + sc.per, (unsigned long long)sc.total);
    if (blockIdx.x == 0 && tid == 0) ws.sched->total = sc.total, ws.sched->per = sc.per;
    const bool find = w0 < w1 && before <= w0 && w0 - before < mine;
    if (find || blockIdx.x == 0) {
        uint32_t at = before;
        for (int s = s_lo; s < s_hi; s++) {
            const uint32_t n = seq_work(c, a, s).units;
            if (blockIdx.x == 0) ws.seq_unit[s] = at;
            if (find && at <= w0 && w0 - at < n) s_seq = s, s_at = at;
            at += n;
        }
    }
    __syncthreads();
    int seq = s_seq;
    uint32_t seq_at = s_at;
    if (seq < 0) return;

    const uint32_t ring = fl_smem_u32(smem) + C::QBYTES + warp * (C::STAGES * C::STAGE);
    const uint8_t* ring_p = smem + C::QBYTES + warp * (C::STAGES * C::STAGE);
    const uint4* q_frag = reinterpret_cast<const uint4*>(smem);
    float* merge = reinterpret_cast<float*>(smem + C::QBYTES);
    SeqWork sw = seq_work(c, a, seq);

    for (uint32_t at = w0; at < w1;) {
        while (at - seq_at >= sw.units) {
            seq_at += sw.units;
            if (++seq >= c.n_seqs) return; /* only where row_start decreases */
            sw = seq_work(c, a, seq);
        }
        /* the segment: tiles [j0, j1) of item (head, row tile) */
        const uint32_t item = (at - seq_at) / sw.cost;
        const uint32_t item_at = seq_at + item * sw.cost + kItemCost;
        const int j0 = at > item_at ? (int)(at - item_at) : 0;
        const int j1 = w1 > item_at ? (int)min((uint32_t)sw.tiles, w1 - item_at) : 0;
        if (j1 <= j0) break; /* the range ends before the item's first tile */
        const int head = (int)item / sw.nrt, rt = (int)item - head * sw.nrt;
        const int f0 = rt * kRows, rows = min(sw.n * a.grp - f0, kRows); /* the item's rows: f0 .. of (row, head of the group) */
        const bool two = rows > 8;
        at = item_at + j1;

        /* ── q fragments ── */
        for (int r = warp; r < kRows; r += kWarps) {
            const int f = f0 + r, i = fl_div_grp(a, f);
            float x[HD / 32];
            uint32_t top = 0;
            if (r < rows) {
                const T* q = static_cast<const T*>(a.q) + (int64_t)(sw.row0 + i) * a.q_stride +
                             (int64_t)(head * a.grp + f - i * a.grp) * HD;
#pragma unroll
                for (int e = 0; e < HD / 32; e++) {
                    x[e] = fl_to_float(q[lane + 32 * e]);
                    top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
                }
                top = __reduce_max_sync(0xffffffffu, top);
                /* q 2^up has its largest magnitude in [2^14, 2^15) */
                const int up = top < 0x7f800000u ? 14 + 127 - (int)(top >> 23) : 0;
                if (lane == 0) s_fr[r] = fl_scale2(a.score_unit, -up);
#pragma unroll
                for (int e = 0; e < HD / 32; e++) x[e] = fl_scale2(x[e], up);
            } else {
#pragma unroll
                for (int e = 0; e < HD / 32; e++) x[e] = 0.0f;
                if (lane == 0) s_fr[r] = 0.0f;
            }
            /* into fragment order: row r of step k, lane (r % 8) * 4 + t, element pairs at words r / 8 and r / 8 + 2 */
#pragma unroll
            for (int e = 0; e < HD / 32; e++) {
                const int d = lane + 32 * e;
                const __half hi = __float2half_rn(x[e]);
                int k, tt;
                if (KV == FL_KV_F16)
                    k = (d >> 5) * 2 + ((d >> 2) & 1), tt = (d >> 3) & 3;
                else
                    k = (d >> 6) * 4 + ((d >> 2) & 3), tt = (d >> 4) & 3;
                __half* dst = reinterpret_cast<__half*>(smem) + (k * 32 + (r & 7) * 4 + tt) * 8 + (r >> 3) * 2 +
                              ((d >> 1) & 1) * 4 + (d & 1);
                dst[0] = hi;
                if (SPLIT) dst[C::KS * 256] = __float2half_rn(x[e] - __half2float(hi));
            }
        }

        /* ── the warp's tiles: j0 + warp, + 4, ..., U at a time ── */
        const int n_mine = j1 - j0 > warp ? (j1 - j0 - warp + kWarps - 1) / kWarps : 0;
        const int tile_first = sw.tile0 + j0 + warp;
        const int32_t* table = c.table + (size_t)seq * c.cols;
        auto page_block = [&](int i0) { /* lane i: the page of the warp's tile i0 + i, or -1 */
            int page = -1;
            if (i0 + lane < n_mine) {
                const int key = (tile_first + (i0 + lane) * kWarps) * kTile;
                if (key < sw.len) page = __ldg(table + (key >> c.page_shift));
                if ((unsigned)page >= (unsigned)c.n_pages) page = -1;
            }
            return page;
        };
        int next_pages = page_block(0), next_block = 0; /* of the tiles being fetched */
        auto fetch = [&](int i) { /* copies of tiles i .. i + U - 1 */
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int x = i + u;
                const uint32_t dst = ring + ((i / U) % C::STAGES) * C::STAGE + u * C::TILE;
                if ((x >> 5) != next_block) {
                    next_block = x >> 5;
                    next_pages = page_block(next_block << 5);
                }
                const int page = __shfl_sync(0xffffffffu, next_pages, x & 31);
                if (page >= 0) {
                    const int key = (tile_first + x * kWarps) * kTile;
                    const int64_t row = (((int64_t)page * c.n_kv + head) << c.page_shift) + (key & ((1 << c.page_shift) - 1));
                    const uint8_t* kp = static_cast<const uint8_t*>(c.k) + row * C::ROW + ((g >> 1) * 4 + (g & 1)) * C::ROW + t * 16;
                    const uint8_t* vp = static_cast<const uint8_t*>(c.v) + row * C::ROW + t * 4 * C::ROW + g * C::VP;
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int p = 0; p < C::KC; p++)
                            fl_cp_async16(dst + (n * C::KC + p) * 512 + lane * 16, kp + n * 2 * C::ROW + p * 64);
#pragma unroll
                    for (int n = 0; n < 4; n++)
#pragma unroll
                        for (int p = 0; p < C::VC; p++) {
                            const uint32_t d = dst + C::KBYTES + (n * C::VC + p) * (32 * C::VP) + lane * C::VP;
                            if (C::VP == 16)
                                fl_cp_async16(d, vp + n * C::ROW + p * 128);
                            else
                                fl_cp_async8(d, vp + n * C::ROW);
                        }
                    if (C::SCALES && lane < 8)
                        fl_cp_async16(dst + 2 * C::KBYTES + lane * 16, (lane < 4 ? c.k_scale : c.v_scale) + row + (lane & 3) * 4);
                } else if (U > 1) {
                    /* computed with its neighbour: zeros, which masked weights keep zero */
#pragma unroll
                    for (int b = 0; b < C::TILE; b += 512)
                        if (b + lane * 16 < C::TILE)
                            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(dst + b + lane * 16), "r"(0) : "memory");
                }
            }
            fl_cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < C::STAGES - 1; i++) fetch(i * U);

        __syncthreads(); /* q fragments */
        uint4 qf[C::QREG ? C::KS : 1], ql[C::QREG && SPLIT ? C::KS : 1];
        if constexpr (C::QREG) {
#pragma unroll
            for (int k = 0; k < C::KS; k++) {
                qf[k] = q_frag[k * 32 + lane];
                if (SPLIT) ql[k] = q_frag[(C::KS + k) * 32 + lane];
            }
        }
        const float fr[2] = {s_fr[g], s_fr[g + 8]};
        int pos[2]; /* last key of rows g, g + 8; rows past the item's see nothing */
#pragma unroll
        for (int i = 0; i < 2; i++) pos[i] = g + 8 * i < rows ? sw.first + fl_div_grp(a, f0 + g + 8 * i) : -1;
        /* the first and the last position of the item's rows */
        const int pos_min = sw.first + fl_div_grp(a, f0), pos_max = sw.first + fl_div_grp(a, f0 + rows - 1);
        const int win = a.window > 0 ? a.window : INT_MAX;

        float acc[C::NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        int ev = -1000; /* exponent of the values' scales that acc counts in (8 bits) */
#pragma unroll
        for (int n = 0; n < C::NT; n++) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;

        int pages = -1;
        for (int i = 0; i < n_mine; i += U) {
            if ((i & 31) == 0) pages = page_block(i);
            fetch(i + (C::STAGES - 1) * U);
            bool mapped[U], any = false;
#pragma unroll
            for (int u = 0; u < U; u++) {
                mapped[u] = __shfl_sync(0xffffffffu, pages, (i + u) & 31) >= 0;
                any |= mapped[u];
            }
            if (any) fl_cp_async_wait<C::STAGES - 1>();
            __syncwarp(); /* scales and zeros are other lanes', and later copies into the place of unread zeros too */
            if (!any) continue;
            const uint8_t* st = ring_p + ((i / U) % C::STAGES) * C::STAGE;
            const int key0 = (tile_first + i * kWarps) * kTile; /* tile u starts at key0 + u * kWarps * kTile */

            /* scores: s[u][n][..] of keys 4t + 2n + {0, 1} of tile u, rows g and g + 8 */
            float s[U][2][4] = {};
#pragma unroll
            for (int p = 0; p < C::KC; p++) {
                uint32_t w[U][2][4];
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const uint4 k4 = *reinterpret_cast<const uint4*>(st + u * C::TILE + (n * C::KC + p) * 512 + lane * 16);
                        w[u][n][0] = k4.x, w[u][n][1] = k4.y, w[u][n][2] = k4.z, w[u][n][3] = k4.w;
                    }
                constexpr int STEPS = KV == FL_KV_F16 ? 2 : 4;
#pragma unroll
                for (int e = 0; e < STEPS; e++) {
                    const int k = p * STEPS + e;
                    const uint4 hi = C::QREG ? qf[C::QREG ? k : 0] : q_frag[k * 32 + lane];
                    const uint4 lo = !SPLIT ? hi : C::QREG ? ql[C::QREG && SPLIT ? k : 0] : q_frag[(C::KS + k) * 32 + lane];
#pragma unroll
                    for (int u = 0; u < U; u++)
#pragma unroll
                        for (int n = 0; n < 2; n++) {
                            uint32_t b0, b1;
                            if constexpr (KV == FL_KV_F16)
                                b0 = w[u][n][2 * e], b1 = w[u][n][2 * e + 1];
                            else
                                fl_widen4<KV>(w[u][n][e], b0, b1);
                            if constexpr (SPLIT) {
                                mma_f16_add(s[u][n], lo, hi, b0, b1);
                            } else {
                                mma_f16(s[u][n], hi, b0, b1);
                            }
                        }
                }
            }
            float sv[U][4];
            bool masked = false; /* some row does not see some key */
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int ku = key0 + u * kWarps * kTile;
                masked |= !mapped[u] || ku + kTile - 1 > pos_min || ku + kTile > sw.len || pos_max - ku >= win;
                if constexpr (C::SCALES != 0) {
                    const float4 k4 = reinterpret_cast<const float4*>(st + u * C::TILE + 2 * C::KBYTES)[t];
                    const float4 v4 = reinterpret_cast<const float4*>(st + u * C::TILE + 2 * C::KBYTES + 64)[t];
                    s[u][0][0] *= k4.x, s[u][0][2] *= k4.x, s[u][0][1] *= k4.y, s[u][0][3] *= k4.y;
                    s[u][1][0] *= k4.z, s[u][1][2] *= k4.z, s[u][1][1] *= k4.w, s[u][1][3] *= k4.w;
                    sv[u][0] = v4.x, sv[u][1] = v4.y, sv[u][2] = v4.z, sv[u][3] = v4.w;
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[u][n][e] *= fr[e >> 1];
            if (a.softcap > 0.0f) {
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (e < 2 || two) s[u][n][e] = tanhf(s[u][n][e]) * (a.softcap * 1.44269504f);
            }
            if (masked) {
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int key = key0 + u * kWarps * kTile + 4 * t + 2 * n + e;
                            const bool there = mapped[u] && key < sw.len;
#pragma unroll
                            for (int i2 = 0; i2 < 2; i2++)
                                if (!(there && key <= pos[i2] && pos[i2] - key < win)) s[u][n][2 * i2 + e] = -INFINITY;
                            /* a scale that no row uses does not count */
                            if (C::SCALES && !(there && key <= pos_max && pos_min - key < win)) sv[u][2 * n + e] = 0.0f;
                        }
            }
            /* running maximum; the exponent of the values' scales likewise */
            float alpha[2] = {1.0f, 1.0f};
            bool moved = false;
#pragma unroll
            for (int i2 = 0; i2 < 2; i2++) {
                if (i2 == 1 && !two) break;
                float mx = s[0][0][2 * i2];
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int n = 0; n < 2; n++) mx = fmaxf(mx, fmaxf(s[u][n][2 * i2], s[u][n][2 * i2 + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                if (mx > m[i2]) {
                    alpha[i2] = fl_ex2(m[i2] - mx); /* 0 the first time */
                    m[i2] = mx;
                    moved = true;
                }
            }
            float up = 16384.0f, down = 1.0f; /* 2^14; what a larger exponent makes of acc */
            if constexpr (C::SCALES != 0) {
                /* the exponent bits of the largest finite scale */
                uint32_t top = 0;
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t b = __float_as_uint(sv[u][e]) & 0x7fffffffu;
                        if (b < 0x7f800000u) top = max(top, b);
                    }
                top = __reduce_max_sync(0xffffffffu, top);
                const int en = max((int)(top >> 23) - 127, -100);
                if (en > ev) {
                    down = ev == -1000 ? 0.0f : fl_ex2((float)(ev - en));
                    ev = en;
                    moved = true;
                }
                up = fl_pow2(14 - ev);
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
            uint4 pa[U], pl[U], seen[U]; /* seen: masked tiles of types with NaN or infinity, 1 where a row sees a key */
#pragma unroll
            for (int u = 0; u < U; u++) {
                uint32_t hi[2][2] = {}, lo[2][2] = {}, se[2][2] = {};
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; e++) f[e] = C::SCALES ? sv[u][e] * up : up;
#pragma unroll
                for (int i2 = 0; i2 < 2; i2++) {
                    if (i2 == 1 && !two) break;
                    const float ref = m[i2] == -INFINITY ? 0.0f : m[i2];
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        float w[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float x = s[u][n][2 * i2 + e], p = fl_ex2(x - ref);
                            l[i2] += p;
                            w[e] = p * f[2 * n + e];
                            if (masked && C::SCALES && x == -INFINITY) w[e] = 0.0f; /* whatever the scale */
                            if (masked && KV != FL_KV_Q8 && x != -INFINITY) se[n][i2] |= 0x3c00u << (16 * e);
                        }
                        hi[n][i2] = fl_pack_half2(w[0], w[1]);
                        if (SPLIT) {
                            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[n][i2]));
                            lo[n][i2] = fl_pack_half2(w[0] - h.x, w[1] - h.y);
                        }
                    }
                }
                pa[u] = make_uint4(hi[0][0], hi[0][1], hi[1][0], hi[1][1]);
                if (SPLIT) pl[u] = make_uint4(lo[0][0], lo[0][1], lo[1][0], lo[1][1]);
                if (KV != FL_KV_Q8) seen[u] = make_uint4(se[0][0], se[0][1], se[1][0], se[1][1]);
            }
            /* values: keys 4t..4t+3 at the lane's elements; tile n of the output holds element n of every lane's run */
#pragma unroll
            for (int pc = 0; pc < C::VC; pc++) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    uint32_t w[4][4];
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const uint8_t* src = st + u * C::TILE + C::KBYTES + (n * C::VC + pc) * (32 * C::VP) + lane * C::VP;
                        if (C::VP == 16) {
                            const uint4 v4 = *reinterpret_cast<const uint4*>(src);
                            w[n][0] = v4.x, w[n][1] = v4.y, w[n][2] = v4.z, w[n][3] = v4.w;
                        } else {
                            const uint2 v2 = *reinterpret_cast<const uint2*>(src);
                            w[n][0] = v2.x, w[n][1] = v2.y;
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
                            fl_widen4<KV>(__byte_perm(w[0][x], w[1][x], 0x5140), b0[0], b0[1]);
                            fl_widen4<KV>(__byte_perm(w[0][x], w[1][x], 0x7362), b0[2], b0[3]);
                            fl_widen4<KV>(__byte_perm(w[2][x], w[3][x], 0x5140), b1[0], b1[1]);
                            fl_widen4<KV>(__byte_perm(w[2][x], w[3][x], 0x7362), b1[2], b1[3]);
                        }
#pragma unroll
                        for (int e = 0; e < PER; e++) {
                            const int n = pc * (C::VP / C::ES) + x * PER + e;
                            if (KV != FL_KV_Q8 && masked) {
                                /* a weight of 0 does not keep NaN or infinity out of a sum: where the tile holds one, it
                                 * is left out, and made NaN in the rows that see it */
                                const uint32_t f0 = odd_halves(b0[e]), f1 = odd_halves(b1[e]);
                                if (__any_sync(0xffffffffu, f0 | f1)) {
                                    float hit[4] = {};
                                    mma_f16(hit, seen[u], f0 & 0x3c003c00u, f1 & 0x3c003c00u);
#pragma unroll
                                    for (int z = 0; z < 4; z++)
                                        if (hit[z] > 0.0f) acc[n][z] = __uint_as_float(0x7fffffffu);
                                    b0[e] &= ~f0;
                                    b1[e] &= ~f1;
                                }
                            }
                            if constexpr (SPLIT) {
                                mma_f16_add(acc[n], pl[u], pa[u], b0[e], b1[e]);
                            } else {
                                mma_f16(acc[n], pa[u], b0[e], b1[e]);
                            }
                        }
                    }
                }
            }
            __syncwarp(); /* the stage's scales are read before another lane's copy may land there */
        }
        fl_cp_async_wait<0>();

        /* ── the CTA's warps, merged in order ── */
#pragma unroll
        for (int i = 0; i < 2; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (t == 0) s_ml[warp][g + 8 * i] = make_float2(m[i], l[i]);
        }
        __syncthreads(); /* every warp is done with its ring, too */
        const int unit = C::SCALES ? (ev == -1000 ? 0 : ev) - 14 : -14;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (i == 1 && !two) break;
            const int r = g + 8 * i;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_ml[w][r].x);
            const float f = m[i] == -INFINITY ? 0.0f : fl_scale2(fl_ex2(m[i] - M), unit);
            float* dst = merge + (warp * kRows + r) * (HD + 4);
            constexpr int RUN = C::VP / C::ES; /* consecutive elements of a lane */
#pragma unroll
            for (int n = 0; n < C::NT; n += 4)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float4 v = make_float4(acc[n][2 * i + e] * f, acc[n + 1][2 * i + e] * f, acc[n + 2][2 * i + e] * f,
                                           acc[n + 3][2 * i + e] * f);
                    if (m[i] == -INFINITY) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    *reinterpret_cast<float4*>(dst + (n / RUN) * 8 * RUN + (2 * t + e) * RUN + n % RUN) = v;
                }
        }
        __syncthreads();
        const bool whole = j0 == 0 && j1 == sw.tiles;
        const int slot = 2 * (int)blockIdx.x + (j0 == 0 ? 1 : 0);
        for (int x = tid; x < rows * (HD / 8); x += kThreads) {
            const int r = x / (HD / 8), d = (x - r * (HD / 8)) * 8;
            float o[8] = {}, M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_ml[w][r].x);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float2 ml = s_ml[w][r];
                L += ml.x == -INFINITY ? ml.y : ml.y * fl_ex2(ml.x - M);
                const float4* src = reinterpret_cast<const float4*>(merge + (w * kRows + r) * (HD + 4) + d);
                const float4 u = src[0], v = src[1];
                o[0] += u.x, o[1] += u.y, o[2] += u.z, o[3] += u.w, o[4] += v.x, o[5] += v.y, o[6] += v.z, o[7] += v.w;
            }
            if (whole) {
                const int f = f0 + r, i = fl_div_grp(a, f), h = head * a.grp + f - i * a.grp;
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

/* Items that several ranges share, a warp per (row, head). */
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) paged_merge_kernel(const FlPaged c, const FlPagedAttn a)
{
    const int64_t pair = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
    if (pair >= (int64_t)c.n_rows * a.n_heads) return fl_pdl_wait(); /* this grid may not end before the one it depends on */
    const int row = (int)((uint32_t)pair / (uint32_t)a.n_heads), h = (int)(pair - (int64_t)row * a.n_heads);
    const int seq = fl_row_seq(c.row_start, c.n_seqs, row);
    if (seq < 0) return fl_pdl_wait();
    const SeqWork sw = seq_work(c, a, seq);
    const int head = fl_div_grp(a, h), f = (row - sw.row0) * a.grp + h - head * a.grp;
    const int item = head * sw.nrt + f / kRows;
    const FlAttnSpace ws = fl_attn_space(a.workspace, c.n_seqs, kMaxCtas, kRows, HD);
    fl_pdl_wait();
    const uint32_t per = ws.sched->per;
    const uint32_t t0 = ws.seq_unit[seq] + (uint32_t)item * sw.cost + kItemCost;
    const int c0 = (int)(t0 / per), c1 = (int)((t0 + sw.tiles - 1) / per);
    if (c0 != c1) fl_merge_row<T, HD>(a, ws, c0, c1, f % kRows, kRows, row, h); /* else written by its range */
}

template <typename T, int KV, int HD>
cudaError_t launch(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    using C = Cfg<KV, HD, sizeof(T) == 4>;
    static_assert(C::CTAS * 148 <= kMaxCtas, "workspace slots");
    static std::atomic<int> sms[64] = {}; /* SMs of a device, once its kernel is configured */
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
    paged_stream_kernel<T, KV, HD><<<sms[dev].load() * C::CTAS, kThreads, C::SMEM, st>>>(c, a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int64_t pairs = (int64_t)c.n_rows * a.n_heads, per_block = kWarps;
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

template <typename T, int HD>
cudaError_t launch_kv(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    switch (c.kv_dtype) {
    case FL_KV_F16: return launch<T, FL_KV_F16, HD>(c, a, st);
    case FL_KV_Q8: return launch<T, FL_KV_Q8, HD>(c, a, st);
    case FL_KV_F8: return launch<T, FL_KV_F8, HD>(c, a, st);
    default: return cudaErrorInvalidValue;
    }
}

template <int HD>
cudaError_t launch_type(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    switch (a.type) {
    case 0: return launch_kv<float, HD>(c, a, st);
    case 1: return launch_kv<__half, HD>(c, a, st);
    case 30: return launch_kv<__nv_bfloat16, HD>(c, a, st);
    default: return cudaErrorInvalidValue;
    }
}

} // namespace
} // namespace flps

#endif
