/*
 * fl_paged_tc.cuh — attention of new rows over a paged KV cache
 * (fl_attn_paged_device) for many query rows per sequence, on the tcgen05
 * tensor cores.  Included by one source file per head dimension.
 *
 * A CTA takes items (sequence, kv head, tile of NQ x 128 query rows, heads of a
 * group folded into the rows) of BK-key tiles, in one contiguous range of the
 * schedule that all items' tiles form, so every SM has the same number of
 * tiles; an item cut by a range's end leaves (o, m, l) in the workspace for a
 * second kernel.  Per key tile:
 *  - 3 warps copy K and V from their pages to shared memory (cp.async); 4 more
 *    make them fp16 in the 128-byte swizzled layout, in place (8-bit elements
 *    are exact in fp16; scales stay beside them), and hand them to the tensor
 *    core.  The two are apart because the fence that hands over waits for every
 *    copy its thread has under way: with both in one thread no tile's copies
 *    overlapped another's work (2048 rows at 16384 keys, 8 bits: 828 us, apart
 *    682 in builds of that time).  V is read by the tensor core with the keys as
 *    its inner dimension, straight from rows of 64 elements (an MN-major operand),
 *    so nothing is transposed.
 *  - one lane issues S = Q K^T into tensor memory and, once the weights are
 *    there, O += P V with P read from tensor memory.
 *  - 4 warps per 128 rows hold one row a thread: S is read from tensor memory
 *    (no shuffles), weights go back as fp16 over the scores.
 * Two sets of scores alternate (two row tiles, or two key tiles where the
 * output takes the room of a second row tile), so the tensor core works on one
 * while the other is exponentiated.  The maximum that weights refer to moves
 * only when it grew by more than 2^8, which leaves O alone on almost every
 * tile; weights then lie below 2^8 and are stored times 2^6, fp16's range.
 *
 * Sums and softmax state are fp32.  32-bit rows use two fp16 for q and for each
 * weight (22 bits) at twice the products.
 *
 * Measured, causal chunk of 2048 rows x 32 heads at the end of 16384 keys, heads
 * of 128: fp16 cache 534 us (965 TFLOP/s of the 1394 that the tensor cores keep
 * up), int8 688 us (749), e4m3 767 us, 32-bit rows over int8 2268 us.  In half of
 * that from fp16 the tensor pipe is busy 39 % of the cycles and the exponentials'
 * 39 %: the 8 softmax warps' own chain, one row a thread (scores out of tensor
 * memory, exponentials, weights back), bounds it; from 8 bits (31 % each) that and
 * the widening through shared memory, which the softmax warps read the scales
 * from.  With softcap (two more transcendental operations a score) 0.2-0.5 k rows at
 * 5 k keys, e4m3, heads of 256: 239 us (caps above 128: 371), of 128: 137 (237).
 */
#ifndef FL_PAGED_TC_CUH
#define FL_PAGED_TC_CUH

#include <atomic>
#include <climits>

#include "fl_paged.cuh"

namespace flpt {
namespace {

constexpr int kSoftWarps = 8, kLoadWarps = 4, kCopyWarps = 3;
constexpr int kThreads = (kSoftWarps + kLoadWarps + 4) * 32; /* the last four: one issues to the tensor core, three copy */
/* registers of a softmax, widening and issuing thread, from the launch's 128 each: a softmax thread holds a row of scores */
constexpr int kSoftRegs = 200, kLoadRegs = 64, kIssueRegs = 48;
static_assert(kSoftWarps * kSoftRegs + kLoadWarps * kLoadRegs + 4 * kIssueRegs <= kThreads / 32 * 128, "register file");
constexpr int kMaxCtas = kFlWaitCtas;
constexpr int kItemCost = 3; /* what starting an item costs, in key tiles */
constexpr int kMinUnits = 2;
constexpr float kLazy = 8.0f; /* log2 of how far weights may exceed 1 */
constexpr int kUp = 6;        /* weights are stored times 2^kUp: below 2^15 with the values' scales below 2 */

template <int KV, int HD, bool SPLIT>
struct Cfg {
    static constexpr int ES = KV == FL_KV_F16 ? 2 : 1;
    static constexpr int ROW = HD * ES;
    static constexpr int NQ = HD == 256 || (SPLIT && HD == 128) ? 1 : 2;
    static constexpr int BK = HD == 256 ? 64 : 128;
    static constexpr int RT = NQ * 128;                    /* query rows of an item */
    static constexpr int STAGES = HD == 64 ? 3 : HD == 256 && SPLIT ? 1 : 2;
    static constexpr int QTILE = 128 * HD * 2;             /* one row tile, one half of the split */
    static constexpr int QBYTES = NQ * QTILE * (SPLIT ? 2 : 1);
    static constexpr int TBYTES = BK * HD * 2;             /* K or V of a key tile */
    static constexpr int PIECES = ROW / 16;                /* 16-byte pieces of a key */
    static constexpr int NP = BK * PIECES / (kLoadWarps * 32); /* pieces of a widening thread */
    /* a piece's place in its tile; an 8-bit one arrives in the first of the two chunks that it widens to */
    static __device__ __forceinline__ uint32_t place(int key, int pc)
    {
        return ES == 2 ? (pc >> 3) * (BK * 128) + key * 128 + (((pc & 7) ^ (key & 7)) << 4)
                       : (pc >> 2) * (BK * 128) + key * 128 + (((pc & 3) * 2 ^ (key & 7)) << 4);
    }
    /* of a key tile: scales of K, of V; (exponent that V's count in, mapped 16-key groups); exponents and findings of the
     * loading warps; values' flags: a byte a key, a bit an element */
    static constexpr int HEAD = BK * 8, EVS = HEAD + 16, BAD = EVS + 32, ODD = BAD + BK, INFO = ODD + BK * HD / 8;
    /* 32-bit rows: key tiles whose products the tensor core sums before the sum is added to one rounded to nearest.  It
     * truncates every sum of 16 products, which always errs towards zero: 5.6 k keys in one run were off by 9.5e-6. */
    static constexpr int RUN = 512 / BK;
    static constexpr int NI = 4;                           /* infos in flight: more than stages, so that they need no release */
    static constexpr int SMEM = QBYTES + STAGES * 2 * TBYTES + NI * INFO + 1024 + 512;
    /* tensor memory columns: two sets of scores (weights over them), the outputs, the weights' low halves */
    static constexpr int S_COL = 0, O_COL = 2 * BK, LOW_COL = 384;
    static_assert(O_COL + NQ * HD <= (SPLIT ? LOW_COL : 512) && SMEM <= 232448, "tensor and shared memory");
};

/* ── the schedule ───────────────────────────────────────────────────────── */
struct SeqWork {
    int row0, n, first, len, nrt;
};
struct ItemWork {
    int f0, rows;            /* folded rows f0 .. f0 + rows - 1 */
    int pos_min, pos_max;    /* positions of the first and the last */
    int tile0, tiles;
};
template <int RT>
__device__ __forceinline__ SeqWork seq_work(const FlPaged& c, const FlPagedAttn& a, int s)
{
    SeqWork w;
    const int r0 = max(__ldg(c.row_start + s), 0), r1 = min(__ldg(c.row_start + s + 1), c.n_rows);
    const int len = fl_seq_len(c, s);
    w.row0 = r0;
    w.n = max(r1 - r0, 0);
    w.first = len - w.n;
    w.len = min(len, c.cols << c.page_shift);
    w.nrt = (w.n * a.grp + RT - 1) / RT;
    return w;
}

template <int RT, int BK>
__device__ __forceinline__ ItemWork item_work(const FlPagedAttn& a, const SeqWork& s, int rt)
{
    ItemWork w;
    w.f0 = rt * RT;
    w.rows = min(s.n * a.grp - w.f0, RT);
    w.pos_min = s.first + fl_div_grp(a, w.f0);
    w.pos_max = s.first + fl_div_grp(a, w.f0 + w.rows - 1);
    const int hi = max(0, min(s.len, w.pos_max + 1));
    w.tile0 = fl_first_seen(w.pos_min, a.window) / BK;
    w.tiles = max(1, (hi + BK - 1) / BK - w.tile0);
    return w;
}

/* Units of one kv head of a sequence's row tiles below `end`. */
template <int RT, int BK>
__device__ __forceinline__ uint32_t head_units(const FlPagedAttn& a, const SeqWork& s, int end)
{
    uint32_t u = 0;
    for (int rt = 0; rt < end; rt++) u += kItemCost + item_work<RT, BK>(a, s, rt).tiles;
    return u;
}

/* ── small helpers ──────────────────────────────────────────────────────── */
/* Keeps sums of x and constants from being formed ahead of a loop and kept in registers. */
__device__ __forceinline__ uint32_t opaque(uint32_t x)
{
    asm volatile("" : "+r"(x));
    return x;
}

/* Two fp32 operations an instruction. */
__device__ __forceinline__ void mul2(float& x0, float& x1, float y0, float y1)
{
    asm("{\n .reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %3};\n mul.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}\n"
        : "+f"(x0), "+f"(x1)
        : "f"(y0), "f"(y1));
}
__device__ __forceinline__ void fma2(float& x0, float& x1, float y, float z)
{
    asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %2};\n mov.b64 c, {%3, %3};\n"
        " fma.rn.f32x2 a, a, b, c;\n mov.b64 {%0, %1}, a;\n}\n"
        : "+f"(x0), "+f"(x1)
        : "f"(y), "f"(z));
}
__device__ __forceinline__ void add2(float& x0, float& x1, float y0, float y1)
{
    asm("{\n .reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %3};\n add.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}\n"
        : "+f"(x0), "+f"(x1)
        : "f"(y0), "f"(y1));
}

__device__ __forceinline__ float recip(float x)
{
    float d;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
    return d;
}
/* tanh y = 1 - 2 / (e^2y + 1), off by some 2^-23 absolutely; below 0.35, where
 * that is too much relatively, the Taylor series to y^11 (the next term is below
 * 2^-26 of the value). */
__device__ __forceinline__ float tanh_of(float y)
{
    const float t = fmaf(-2.0f, recip(fl_ex2(y * 2.88539008f) + 1.0f), 1.0f), z = y * y;
    float p = -1382.0f / 155925.0f;
    p = fmaf(p, z, 62.0f / 2835.0f);
    p = fmaf(p, z, -17.0f / 315.0f);
    p = fmaf(p, z, 2.0f / 15.0f);
    p = fmaf(p, z, -1.0f / 3.0f);
    return fabsf(y) < 0.35f ? fmaf(p * z, y, y) : t;
}

/* One bit per half of w that is NaN or infinite. */
__device__ __forceinline__ uint32_t odd_bits(uint32_t w)
{
    return ((w & 0x7c00u) == 0x7c00u ? 1u : 0u) | ((w & 0x7c000000u) == 0x7c000000u ? 2u : 0u);
}

__device__ __forceinline__ void sts16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w)
{
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
/* Descriptors of 128-byte swizzled tiles: rows of 128 bytes, groups of 8 rows
 * 1024 bytes apart.  As a K-major operand (rows = M or N) the leading offset is
 * unused; as an MN-major one (rows = K) it is the distance to the next 64
 * elements of N.  The low word holds address and leading offset in 16-byte
 * units, the high word group stride, version and swizzle. */
constexpr uint32_t kDescHigh = (1024 >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t tile_desc(uint32_t saddr, uint32_t lbo) { return (saddr & 0x3FFFFu) >> 4 | (lbo >> 4) << 16; }
/* kind::f16, A and B fp16, D fp32, M = 128; bit 16: B is MN-major. */
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn)
{
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, bool accum)
{
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"((uint32_t)accum), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, bool accum)
{
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"((uint32_t)accum), "r"(kDescHigh)
        : "memory");
}
/* Arrives on `bar` once this thread's copies so far have landed. */
__device__ __forceinline__ void copies_arrive(uint64_t* bar)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(fl_smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(fl_smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

/* What sums that count in (m0, e0) are worth where others count in (m, e). */
__device__ __forceinline__ float part_unit(float m0, float m, int e0, int e)
{
    return (m0 == m ? 1.0f : fl_ex2(m0 - m)) * fl_ex2((float)(e0 - e));
}
__device__ __forceinline__ void add_part(const float* part, float unit, float (&v)[32])
{
#pragma unroll
    for (int z = 0; z < 32; z += 4) {
        const float4 p = *reinterpret_cast<const float4*>(part + z);
        v[z] = fmaf(p.x, unit, v[z]), v[z + 1] = fmaf(p.y, unit, v[z + 1]);
        v[z + 2] = fmaf(p.z, unit, v[z + 2]), v[z + 3] = fmaf(p.w, unit, v[z + 3]);
    }
}

#define FL_F32(c, v) \
    c(v[0]), c(v[1]), c(v[2]), c(v[3]), c(v[4]), c(v[5]), c(v[6]), c(v[7]), c(v[8]), c(v[9]), c(v[10]), c(v[11]), c(v[12]), \
        c(v[13]), c(v[14]), c(v[15]), c(v[16]), c(v[17]), c(v[18]), c(v[19]), c(v[20]), c(v[21]), c(v[22]), c(v[23]), \
        c(v[24]), c(v[25]), c(v[26]), c(v[27]), c(v[28]), c(v[29]), c(v[30]), c(v[31])
/* 32 consecutive columns of the thread's lane; to be used after tmem_wait_ld on them. */
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : FL_F32("=f", v)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(float* v)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : FL_F32("+f", v)::"memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float* v)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        FL_F32("f", v)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

/* The warps of a role. */
__device__ __forceinline__ void role_sync(int role)
{
    asm volatile("bar.sync %0, %1;" ::"r"(role + 1), "r"(role == 4 ? kCopyWarps * 32 : 128) : "memory");
}

/* Barriers that tell whether any thread passed `bad`: of a role, of the softmax warps. */
__device__ __forceinline__ bool bar_any(int id, int threads, bool bad)
{
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n bar.red.or.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(r)
        : "r"(id), "r"(threads), "r"((uint32_t)bad)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ bool role_any(int role, bool bad) { return bar_any(role + 1, role == 4 ? kCopyWarps * 32 : 128, bad); }
__device__ __forceinline__ bool pair_any(bool bad) { return bar_any(8, kSoftWarps * 32, bad); }

/* Bounded wait (~2 s); false once it ran out or another role of the CTA gave up. */
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort)
{
    if (fl_mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = fl_globaltimer();
    for (uint32_t it = 1;; it++) {
        if (fl_mbar_try_wait(bar, parity)) return true;
        if ((it & 1023u) == 0) {
            if (*abort) return false;
            if (fl_globaltimer() - t0 > 2000000000ull) {
                *abort = 1;
                return false;
            }
        }
    }
}

/* *to = *flag, 0 or 1.  Written in C it had the register allocator spill in the softmax loop of the folded softcap (heads
 * of 256, e4m3: 238 -> 250 us). */
__device__ __forceinline__ void copy_flag(uint8_t* to, volatile int* flag)
{
    asm volatile("{\n .reg .u32 t;\n ld.volatile.shared.u32 t, [%0];\n st.global.u8 [%1], t;\n}\n" ::"r"(
                     fl_smem_u32(const_cast<int*>(flag))),
                 "l"(to)
                 : "memory");
}

/* The same for a whole warp, which stays together. */
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort)
{
    return __all_sync(0xffffffffu, wait_bar(bar, parity, abort));
}

/* Where a range stands: iterates the segments (items cut to the range) in the
 * same way in every role.  Each role keeps one in shared memory, moved on by
 * one of its threads, so that its state takes no registers in the loops. */
template <int RT, int BK>
struct Segments {
    uint32_t at, end, seq_at, head_u;
    int seq;
    SeqWork sw;
    /* of the current segment */
    ItemWork it;
    int head, rt, j0, j1;
    bool more;

    __device__ __forceinline__ void enter(const FlPaged& c, const FlPagedAttn& a, int s)
    {
        seq = s;
        sw = seq_work<RT>(c, a, s);
        head_u = head_units<RT, BK>(a, sw, sw.nrt);
    }
    __device__ __forceinline__ bool next(const FlPaged& c, const FlPagedAttn& a)
    {
        while (at < end) {
            while (at - seq_at >= head_u * c.n_kv) {
                seq_at += head_u * c.n_kv;
                if (seq + 1 >= c.n_seqs) { /* only where row_start decreases */
                    at = end;
                    return false;
                }
                enter(c, a, seq + 1);
            }
            uint32_t off = at - seq_at;
            head = (int)(off / head_u);
            off -= head * head_u;
            uint32_t item_at = at - off;
            for (rt = 0;; rt++) {
                it = item_work<RT, BK>(a, sw, rt);
                const uint32_t n = kItemCost + it.tiles;
                if (off < n) break;
                off -= n;
                item_at += n;
            }
            item_at += kItemCost;
            j0 = at > item_at ? (int)(at - item_at) : 0;
            j1 = end > item_at ? (int)min((uint32_t)it.tiles, end - item_at) : 0;
            at = item_at + it.tiles;
            if (at > end) at = end;
            if (j1 > j0) return true;
        }
        return false;
    }
};

/* Softcap's variants, each of its own because 128 curves at once cost the plain
 * kernel registers that it does not have to spare: kCapFolded joins the curve to
 * the weights' multiply and add, off by some 2^-22 of the cap, which up to kFoldMax
 * is at most 2^-15 of a weight, a sixteenth of the rounding of one to fp16;
 * kCapCurve, for larger caps and for 32-bit rows, is off by some 2^-21 of the score
 * (three chunks of 0.2-0.5 k rows, e4m3, heads of 256: 239 and 371 us, of 128: 137
 * and 237). */
constexpr int kNoCap = 0, kCapFolded = 1, kCapCurve = 2;
constexpr float kFoldMax = 128.0f;
template <typename T, int KV, int HD, int CAP>
__global__ void __launch_bounds__(kThreads, 1) paged_tc_kernel(const FlPaged c, const FlPagedAttn a)
{
    constexpr bool SPLIT = sizeof(T) == 4;
    using C = Cfg<KV, HD, SPLIT>;
    constexpr int NQ = C::NQ, BK = C::BK, ST = C::STAGES, RT = C::RT;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = fl_smem_u32(smem_raw), s_base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (s_base - raw);
    const uint32_t s_q = s_base, s_k = s_base + C::QBYTES, s_v = s_k + ST * C::TBYTES;
    uint8_t* info = smem + C::QBYTES + 2 * ST * C::TBYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(info + C::NI * C::INFO);
    uint64_t *k_full = bars, *k_empty = bars + 3, *v_full = bars + 6, *v_empty = bars + 9;
    uint64_t *s_full = bars + 12, *p_full = bars + 14, *q_full = bars + 16, *o_full = bars + 17, *pv_done = bars + 18,
             *done = bars + 19, *i_full = bars + 20,
             *k_raw = bars + 24, *v_raw = bars + 27;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 30);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_holder + 1);
    __shared__ uint32_t s_scan[kThreads / 32], s_at;
    __shared__ int s_seq;
    __shared__ float s_fr[RT];                    /* score units of a row's scaled q */
    __shared__ Segments<RT, BK> s_seg[5];
    __shared__ uint32_t s_nan[256][HD / 32]; /* elements of a row's output that are NaN, as a softmax thread found them */
    /* one row tile: what the two threads of a row tell each other */
    constexpr bool PAIR = NQ == 1;
    __shared__ float2 s_ref[PAIR ? 128 : 1];      /* maximum and exponent of the last tile so far */
    __shared__ float4 s_end[2][PAIR ? 128 : 1];   /* at a segment's end: l, its maximum, flags, kept sums' maximum */
    __shared__ int s_end_e[PAIR ? 128 : 1];       /* and their exponent */
    __shared__ uint64_t s_turn[2][4];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const FlAttnSpace ws = fl_attn_space(a.workspace, c.n_seqs, kMaxCtas, RT, HD);
    fl_pdl_trigger(); /* the merge kernel may take its place; it waits for this grid's end */

    if (tid == 0) {
        for (int s = 0; s < 3; s++) {
            fl_mbar_init(&k_full[s], kLoadWarps * 32);
            fl_mbar_init(&v_full[s], kLoadWarps * 32);
            fl_mbar_init(&k_empty[s], 1);
            fl_mbar_init(&v_empty[s], 1);
            /* each copying thread arrives twice: by its copies, and for its own stores */
            fl_mbar_init(&k_raw[s], 2 * kCopyWarps * 32);
            fl_mbar_init(&v_raw[s], 2 * kCopyWarps * 32);
        }
        for (int i = 0; i < C::NI; i++) fl_mbar_init(&i_full[i], kLoadWarps * 32);
        for (int b = 0; b < 2; b++) {
            fl_mbar_init(&s_full[b], 1);
            fl_mbar_init(&p_full[b], 4);
        }
        fl_mbar_init(q_full, kSoftWarps);
        for (int i = 0; i < 8; i++) fl_mbar_init(&s_turn[i >> 2][i & 3], 1);
        fl_mbar_init(o_full, 1);
        fl_mbar_init(pv_done, 1);
        fl_mbar_init(done, 1);
        *abort = 0;
        s_seq = -1;
        fl_fence_mbar_init();
    }
    if (warp == kSoftWarps + kLoadWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(fl_smem_u32(tmem_holder)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    /* ── this CTA's range: a scan over the sequences' units ── */
    const int per_thread = (c.n_seqs + kThreads - 1) / kThreads;
    const int lo = min(tid * per_thread, c.n_seqs), hi = min(lo + per_thread, c.n_seqs);
    auto units = [&](int s) {
        const SeqWork w = seq_work<RT>(c, a, s);
        return head_units<RT, BK>(a, w, w.nrt) * (uint32_t)c.n_kv;
    };
    uint32_t mine = 0;
    for (int s = lo; s < hi; s++) mine += units(s);
    uint32_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += u;
    }
    if (lane == 31) s_scan[warp] = before;
    fence_before();
    __syncthreads();
    fence_after();
    struct {
        uint32_t total, per;
    } sc;
    sc.total = 0;
    before -= mine;
    for (int w = 0; w < kThreads / 32; w++) {
        if (w < warp) before += s_scan[w];
        sc.total += s_scan[w];
    }
    sc.per = max((uint32_t)kMinUnits, (sc.total + gridDim.x - 1) / gridDim.x);
    const unsigned long long w0_64 = (unsigned long long)blockIdx.x * sc.per;
    const uint32_t range_lo = (uint32_t)min(w0_64, (unsigned long long)sc.total);
    const uint32_t range_hi = (uint32_t)min(w0_64 + sc.per, (unsigned long long)sc.total);
    if (blockIdx.x == 0 && tid == 0) ws.sched->total = sc.total, ws.sched->per = sc.per;
    const bool find = range_lo < range_hi && before <= range_lo && range_lo - before < mine;
    if (find || blockIdx.x == 0) {
        uint32_t at = before;
        for (int s = lo; s < hi; s++) {
            const uint32_t n = units(s);
            if (blockIdx.x == 0) ws.seq_unit[s] = at;
            if (find && at <= range_lo && range_lo - at < n) s_seq = s, s_at = at;
            at += n;
        }
    }
    __syncthreads();
    const uint32_t tmem = *tmem_holder;
    const bool work = s_seq >= 0;
    /* roles: softmax of row tile 0, of row tile 1, widening, issuing, copying */
    const int role = warp <= kSoftWarps + kLoadWarps ? warp >> 2 : 4;
    const bool leads = role == 4 ? tid == kThreads - kCopyWarps * 32 : (tid & 127) == 0;
    Segments<RT, BK>& seg = s_seg[role];
    if (work && leads) {
        seg.at = range_lo;
        seg.end = range_hi;
        seg.seq_at = s_at;
        seg.enter(c, a, s_seq);
    }
    /* the next segment, for all warps of a role; none once a wait of one of them ran out */
    auto next_segment = [&](bool ok) {
        if (role_any(role, !ok)) return false;
        if (leads) seg.more = seg.next(c, a);
        role_sync(role);
        return seg.more;
    };
    const int win = a.window > 0 ? a.window : INT_MAX;

    if (!work) {
    } else if (warp >= kSoftWarps && warp < kSoftWarps + kLoadWarps) {
        /* ── K and V as the tensor core reads them ── */
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
        const int lt = tid - kSoftWarps * 32;
        constexpr int KPP = kLoadWarps * 32 / C::PIECES; /* keys that a pass of the warps covers */
        /* 8-bit: eight lanes hold four pieces of two keys, whose stores of 32 bytes a piece then lie on different banks */
        const int pc = C::ES == 2 ? lt % C::PIECES : (lane & 3) | ((lane >> 3) * 4) % C::PIECES;
        const int k_in = C::ES == 2 ? lt / C::PIECES : (warp & 3) * (32 / C::PIECES) + (lane >> 3) * 4 / C::PIECES * 2 + ((lane >> 2) & 1);
        int n = 0; /* key tiles so far */
        bool ok = true;
        while (next_segment(ok)) {
            const int pos_min = seg.it.pos_min, pos_max = seg.it.pos_max;
            const int see_lo = fl_first_seen(pos_min, a.window); /* keys that some row sees */
            const int see_hi = min(seg.sw.len, pos_max + 1);
            const int key_end = (seg.it.tile0 + seg.j1) * BK;
            int e_run = -100;
            auto widen = [&](uint32_t base) { /* this thread's pieces of a tile, each in the two chunks that are its own */
                if constexpr (C::ES == 1) {
                    const uint32_t to = opaque(base + C::place(k_in, pc));
#pragma unroll
                    for (int i0 = 0; i0 < C::NP; i0 += 4) { /* four loads under way at once */
                        uint4 r[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) r[i] = lds16(to + (i0 + i) * (KPP * 128));
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t at = to + (i0 + i) * (KPP * 128), w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
                            uint32_t h[8];
#pragma unroll
                            for (int x = 0; x < 4; x++) fl_widen4<KV>(w[x], h[2 * x], h[2 * x + 1]);
                            sts16(at, h[0], h[1], h[2], h[3]);
                            sts16(at ^ 16u, h[4], h[5], h[6], h[7]);
                        }
                    }
                }
            };
            for (int key0 = (seg.it.tile0 + seg.j0) * BK; key0 < key_end; key0 += BK, n++) {
                const int st = n % ST;
                const uint32_t par = (n / ST) & 1;
                uint8_t* inf = info + (n % C::NI) * C::INFO;
                int* evs = reinterpret_cast<int*>(inf + C::EVS);
                const uint32_t vd = s_v + st * C::TBYTES;
                const bool partial = key0 + BK - 1 > pos_min || pos_max - key0 >= win;
                if (!(ok = wait_warp(&k_raw[st], par, abort))) break;
                if constexpr (C::ES == 1) {
                    /* V's scales; the largest finite one's exponent, so far in this segment */
                    float sv = 0.0f;
                    if (lt < BK && key0 + lt >= see_lo && key0 + lt < see_hi) sv = reinterpret_cast<const float*>(inf)[BK + lt];
                    const uint32_t b = __float_as_uint(sv) & 0x7fffffffu;
                    const uint32_t top = __reduce_max_sync(0xffffffffu, b < 0x7f800000u ? b : 0u);
                    if (lane == 0) evs[warp & 3] = (int)(top >> 23) - 127;
                    if (partial && lt < BK) { /* a scale that is no number counts as the row's elements would */
                        const bool bad = b >= 0x7f800000u;
                        (inf + C::BAD)[lt] = bad;
                        if (bad) sv = 0.0f;
                    }
                    role_sync(2);
                    e_run = max(e_run, max(max(evs[0], evs[1]), max(evs[2], evs[3])));
                    if (lt < BK) reinterpret_cast<float*>(inf)[BK + lt] = fl_scale2(sv, kUp - e_run);
                }
                if (lt == 0) *reinterpret_cast<int*>(inf + C::HEAD) = e_run;
                fl_mbar_arrive(&i_full[n % C::NI]);
                widen(s_k + st * C::TBYTES);
                fl_fence_proxy_async();
                fl_mbar_arrive(&k_full[st]);
                if (!(ok = wait_warp(&v_raw[st], par, abort))) break;
                if (partial) {
                    /* keys that no row sees become zero; NaN and infinities that only some rows see are noted and left out */
                    bool any = false;
#pragma unroll 1
                    for (int i = 0; i < C::NP; i++) {
                        const int kk = i * KPP + k_in;
                        const uint32_t at = vd + C::place(kk, pc);
                        uint32_t bits = 0;
                        if (key0 + kk < see_lo || key0 + kk >= see_hi) {
                            sts16(at, 0, 0, 0, 0);
                        } else if (KV != FL_KV_Q8) {
                            const uint4 v = lds16(at);
                            uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int x = 0; x < 4; x++) {
                                uint32_t b, gone;
                                if (KV == FL_KV_F16) {
                                    b = odd_bits(w[x]);
                                    gone = (b & 1 ? 0xffffu : 0u) | (b & 2 ? 0xffff0000u : 0u);
                                } else { /* 0x7f is e4m3's NaN */
                                    gone = __vcmpeq4(w[x] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                                    b = (gone & 1u) | (gone >> 8 & 1u) << 1 | (gone >> 16 & 1u) << 2 | (gone >> 24 & 1u) << 3;
                                }
                                bits |= b << (x * (16 / C::ES / 4));
                                w[x] &= ~gone;
                            }
                            if (bits) sts16(at, w[0], w[1], w[2], w[3]);
                        }
                        if (C::ES == 1) {
                            if ((inf + C::BAD)[kk]) bits = 0xffffu;
                            reinterpret_cast<uint16_t*>(inf + C::ODD)[kk * (HD / 16) + pc] = (uint16_t)bits;
                        } else {
                            (inf + C::ODD)[kk * (HD / 8) + pc] = (uint8_t)bits;
                        }
                        any |= bits != 0;
                    }
                    any = __any_sync(0xffffffffu, any);
                    if (lane == 0) evs[4 + (warp & 3)] = any;
                }
                widen(vd);
                fl_fence_proxy_async();
                fl_mbar_arrive(&v_full[st]);
            }
        }
    } else if (warp >= kSoftWarps + kLoadWarps) {
        /* ── the tensor core ── */
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (role == 4) {
            /* ── copies out of the pages ── */
            constexpr int KI = 32 / C::PIECES; /* keys that a warp copies at once */
            const int ct = tid - (kThreads - kCopyWarps * 32);
            const uint32_t mine = C::place(lane / C::PIECES, lane % C::PIECES);
            int n = 0;
            bool ok = !a.stall;
            while (next_segment(ok)) {
                const int32_t* table = c.table + (size_t)seg.seq * c.cols;
                const int see_hi = min(seg.sw.len, seg.it.pos_max + 1), head = seg.head, in_page = (1 << c.page_shift) - 1;
                const int key_end = (seg.it.tile0 + seg.j1) * BK;
                auto pages_of = [&](int k0) { /* lane i: the table's entry for keys k0 + 16 i .., unchecked so that nothing waits for it */
                    int page = -1;
                    const int key = k0 + 16 * lane;
                    if (lane < BK / 16 && key < see_hi && k0 < key_end) page = __ldg(table + (key >> c.page_shift));
                    return page;
                };
                int key0 = (seg.it.tile0 + seg.j0) * BK, next_page = pages_of(key0);
                for (; key0 < key_end; key0 += BK, n++) {
                    const int page = next_page, st = n % ST;
                    const uint32_t par = ((n / ST) & 1) ^ 1;
                    uint8_t* inf = info + (n % C::NI) * C::INFO;
                    next_page = pages_of(key0 + BK);
                    auto row_of = [&](int kk) -> int64_t { /* cache row of key key0 + kk; -1: unmapped */
                        const int pg = __shfl_sync(0xffffffffu, page, kk >> 4);
                        if ((unsigned)pg >= (unsigned)c.n_pages) return -1;
                        return (((int64_t)pg * c.n_kv + head) << c.page_shift) + ((key0 + kk) & in_page);
                    };
                    auto bring = [&](uint32_t base, const void* src, uint64_t* bar) {
                        /* a warp takes 16 keys, which lie in one page and in a row, lane by lane 16 bytes */
                        for (int grp = ct >> 5; grp < BK / 16; grp += kCopyWarps) {
                            const int64_t row = row_of(grp * 16);
                            const uint8_t* from = static_cast<const uint8_t*>(src) + row * C::ROW + lane * 16;
                            const uint32_t to = base + grp * (16 * 128);
                            if (row >= 0) {
#pragma unroll
                                for (int i = 0; i < C::PIECES / 2; i++)
                                    fl_cp_async16(to + i * KI * 128 + (mine ^ ((i * KI & 7) << 4)), from + i * 512);
                            } else {
#pragma unroll
                                for (int i = 0; i < C::PIECES / 2; i++)
                                    sts16(to + i * KI * 128 + (mine ^ ((i * KI & 7) << 4)), 0, 0, 0, 0);
                            }
                        }
                        copies_arrive(bar);
                        fl_mbar_arrive(bar);
                    };
                    if (!(ok = wait_warp(&k_empty[st], par, abort))) break;
                    const uint32_t mapped = __ballot_sync(0xffffffffu, (unsigned)page < (unsigned)c.n_pages) & ((1u << (BK / 16)) - 1);
                    if (ct == 0) *reinterpret_cast<int*>(inf + C::HEAD + 4) = (int)mapped;
                    if constexpr (C::ES == 1) { /* scales of K, then of V: four a piece */
                        const int kk = (ct & (BK / 4 - 1)) * 4;
                        const int64_t row = row_of(kk);
                        if (ct < BK / 2) {
                            const bool v = ct >= BK / 4;
                            const uint32_t to = fl_smem_u32(inf) + (v ? BK * 4 : 0) + kk * 4;
                            if (row >= 0)
                                fl_cp_async16(to, (v ? c.v_scale : c.k_scale) + row);
                            else
                                sts16(to, 0, 0, 0, 0);
                        }
                    }
                    bring(s_k + st * C::TBYTES, c.k, &k_raw[st]);
                    if (!(ok = wait_warp(&v_empty[st], par, abort))) break;
                    bring(s_v + st * C::TBYTES, c.v, &v_raw[st]);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else if (lane == 0) {
            constexpr uint32_t id_s = idesc(BK, false), id_o = idesc(HD, true);
            constexpr int H = SPLIT ? 2 : 1;
            bool ok = true;
            int n = 0;
            uint32_t segs = 0, p_ph = 0; /* phases: bit b of p_ph for weights b */
            auto scores = [&](int q, int buf, int st) { /* S[buf] = Q_q K^T */
                const uint32_t d = opaque(tmem + C::S_COL + buf * BK);
                const uint32_t qd = opaque(tile_desc(s_q + q * H * C::QTILE, 16)), kd = opaque(tile_desc(s_k + st * C::TBYTES, 16));
#pragma unroll
                for (int h = H - 1; h >= 0; h--) /* the low half first */
#pragma unroll
                    for (int k = 0; k < HD / 16; k++)
                        umma_ss(d, qd + h * (C::QTILE >> 4) + (k >> 2) * (16384 >> 4) + (k & 3) * 2,
                                kd + (k >> 2) * (BK * 128 >> 4) + (k & 3) * 2, id_s, h != H - 1 || k != 0);
                umma_commit(&s_full[buf]);
            };
            auto values = [&](int q, int buf, int st, bool more) { /* O_q (+)= P[buf] V */
                const uint32_t d = opaque(tmem + C::O_COL + q * HD), p = opaque(tmem + C::S_COL + buf * BK);
                const uint32_t vd = opaque(tile_desc(s_v + st * C::TBYTES, BK * 128)), low = opaque(tmem + C::LOW_COL + buf * (BK / 2));
#pragma unroll
                for (int h = H - 1; h >= 0; h--)
#pragma unroll
                    for (int k = 0; k < BK / 16; k++)
                        umma_ts(d, (h ? low : p) + k * 8, vd + k * (2048 >> 4), id_o,
                                more || h != H - 1 || k != 0);
            };
            for (;;) {
                seg.more = seg.next(c, a);
                if (!seg.more) break;
                const int tiles = seg.j1 - seg.j0, nq = NQ == 2 && seg.it.rows > 128 ? 2 : 1;
                if (!(ok = wait_bar(q_full, segs & 1, abort))) break;
                if (!(ok = wait_bar(&k_full[n % ST], (n / ST) & 1, abort))) break;
                fence_after();
                for (int q = 0; q < nq; q++) scores(q, q, n % ST);
                umma_commit(&k_empty[n % ST]);
                for (int j = 0; j < tiles && ok; j++) {
                    const int sv = (n + j) % ST, sk = (n + j + 1) % ST;
                    const uint32_t v_par = ((n + j) / ST) & 1, k_par = ((n + j + 1) / ST) & 1;
                    const bool more = j + 1 < tiles;
                    if (NQ == 1 && ST > 1 && more) { /* the next scores while these are exponentiated */
                        if (!(ok = wait_bar(&k_full[sk], k_par, abort))) break;
                        fence_after();
                        scores(0, (j + 1) & 1, sk);
                        umma_commit(&k_empty[sk]);
                    }
                    if (!(ok = wait_bar(&v_full[sv], v_par, abort))) break;
                    for (int q = 0; q < nq; q++) {
                        const int buf = NQ == 1 ? j & 1 : q;
                        if (!(ok = wait_bar(&p_full[buf], (p_ph >> buf) & 1, abort))) break;
                        p_ph ^= 1u << buf;
                        fence_after();
                        values(q, buf, sv, SPLIT ? (j & (C::RUN - 1)) != 0 : j > 0);
                        if (NQ == 1) umma_commit(pv_done);
                        if (NQ == 2 && more) {
                            if (q == 0 && !(ok = wait_bar(&k_full[sk], k_par, abort))) break;
                            fence_after();
                            scores(q, q, sk);
                        }
                    }
                    umma_commit(&v_empty[sv]);
                    if (NQ == 2 && more) umma_commit(&k_empty[sk]);
                    if (NQ == 1 && ST == 1 && more) { /* one stage: the next keys come once these values are done */
                        if (!(ok = wait_bar(&k_full[sk], k_par, abort))) break;
                        fence_after();
                        scores(0, (j + 1) & 1, sk);
                        umma_commit(&k_empty[sk]);
                    }
                }
                if (!ok) break;
                umma_commit(o_full);
                n += tiles;
                segs++;
            }
            /* every product issued is done before the tensor memory is freed */
            umma_commit(done);
            const bool dummy = fl_mbar_wait(done, 0, nullptr);
            (void)dummy;
        }
    } else {
        /* ── softmax: a row per thread ── */
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        const int q = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        /* One row tile: the two warps of 32 rows take its key tiles in turn.  A tile's scores are fetched, scaled, curved
         * and searched for their maximum beside the other warp's exponentials; only the reference goes from one to the
         * other, tile by tile. */
        const int mine_q = PAIR ? 0 : q, row = mine_q * 128 + r;
        int n0 = 0; /* tiles of the segments before */
        uint32_t segs = 0, s_ph = 0, pv_ph = 0, turns = 0; /* phases: bit b of s_ph for scores b; turns: of the other warp */
        bool ok = true;
        while (next_segment(ok)) {
            const int tiles = seg.j1 - seg.j0;
            const bool live = PAIR || q == 0 || seg.it.rows > 128; /* a second row tile may be empty */
            /* q of this warp's 32 rows, as fp16 of largest magnitude in [2^14, 2^15) */
            {
                constexpr int LANES = HD / 8, PER = 32 / LANES;
#pragma unroll 2
                for (int x = PAIR ? q * 16 : 0; x < (PAIR ? q * 16 + 16 : 32); x += PER) {
                    const int row = mine_q * 128 + quarter * 32 + x + lane / LANES, e = (lane % LANES) * 8;
                    float v[8] = {};
                    if (row < seg.it.rows) {
                        const int f = seg.it.f0 + row, i = fl_div_grp(a, f);
                        fl_load8(static_cast<const T*>(a.q) + (int64_t)(seg.sw.row0 + i) * a.q_stride +
                                     (int64_t)(seg.head * a.grp + f - i * a.grp) * HD + e, v);
                    }
                    uint32_t top = 0;
#pragma unroll
                    for (int z = 0; z < 8; z++) top = max(top, __float_as_uint(v[z]) & 0x7fffffffu);
#pragma unroll
                    for (int o = 1; o < LANES; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const int up = top < 0x7f800000u ? min(14 + 127 - (int)(top >> 23), a.up_max) : 0;
                    if (e == 0) s_fr[row] = fl_scale2(a.unit, -up);
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int z = 0; z < 4; z++) {
                        const float y0 = fl_scale2(v[2 * z], up) * a.q_sign, y1 = fl_scale2(v[2 * z + 1], up) * a.q_sign;
                        h[z] = fl_pack_half2(y0, y1);
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[z]));
                        l[z] = fl_pack_half2(y0 - f.x, y1 - f.y);
                    }
                    const int rr = quarter * 32 + x + lane / LANES;
                    const uint32_t at = s_q + mine_q * (SPLIT ? 2 : 1) * C::QTILE + (e >> 6) * 16384 + rr * 128 +
                                        ((((e >> 3) & 7) ^ (rr & 7)) << 4);
                    sts16(at, h[0], h[1], h[2], h[3]);
                    if (SPLIT) sts16(at + C::QTILE, l[0], l[1], l[2], l[3]);
                }
                fl_fence_proxy_async();
                __syncwarp();
                if (lane == 0) fl_mbar_arrive(q_full);
                /* Every warp waits for the others' rows, those of an empty row tile too, which have nothing else to wait
                 * for: without it they would arrive for later items in place of the warps that still read this one's. */
                ok = wait_warp(q_full, segs & 1, abort);
            }
            const float fr = s_fr[row];
            const int pos = row < seg.it.rows ? seg.sw.first + fl_div_grp(a, seg.it.f0 + row) : -1;
            const int pos_min = seg.it.pos_min, pos_max = seg.it.pos_max, len = seg.sw.len;
            const int key_first = (seg.it.tile0 + seg.j0) * BK;
            float m = -INFINITY, l = 0.0f;
            int e_acc = -100; /* exponent of the values' scales that O counts in */
            bool any_nan = false;
            /* where the item's sums are kept: its partial result's place, which is this CTA's */
            const int slot = 2 * (int)blockIdx.x + (seg.j0 == 0 ? 1 : 0);
            float* part = ws.o + ((size_t)slot * RT + row) * HD;
            float m_part = 0.0f; /* the maximum and the exponent that they count in */
            int e_part = 0;
            for (int j = PAIR ? q : 0; ok && j < tiles; j += PAIR ? 2 : 1) {
                const int n = n0 + j, key0 = key_first + j * BK, st = n % ST, buf = q;
                const uint8_t* inf = info + (n % C::NI) * C::INFO;
                if (!live) continue;
                if (!(ok = wait_warp(&i_full[n % C::NI], (n / C::NI) & 1, abort))) break;
                if (!(ok = wait_warp(&s_full[buf], (s_ph >> buf) & 1, abort))) break;
                s_ph ^= 1u << buf;
                fence_after();
                const uint32_t s_at = lanes + C::S_COL + buf * BK;
                const float* sk = reinterpret_cast<const float*>(inf);
                const float* sv = sk + BK;
                const int* evs = reinterpret_cast<const int*>(inf + C::EVS);
                const int2 head = *reinterpret_cast<const int2*>(inf + C::HEAD);
                const bool holes = head.y != (1 << (BK / 16)) - 1;
                const bool partial = key0 + BK - 1 > pos_min || pos_max - key0 >= win;
                /* columns the row sees: (c_lo, c_hi] */
                const int c_hi = min(pos, len - 1) - key0, c_lo = pos - key0 < win ? -1 : pos - key0 - win;
                float x[BK];
#pragma unroll
                for (int b = 0; b < BK; b += 32) tmem_ld32(s_at + b, x + b);
#pragma unroll
                for (int b = 0; b < BK; b += 32) tmem_wait_ld(x + b);
                if (C::ES == 1) {
#pragma unroll
                    for (int z = 0; z < BK; z += 4) {
                        const float4 k4 = *reinterpret_cast<const float4*>(sk + z);
                        mul2(x[z], x[z + 1], k4.x, k4.y);
                        mul2(x[z + 2], x[z + 3], k4.z, k4.w);
                    }
                }
                auto mask = [&](float unseen) {
                    const uint32_t seen = (uint32_t)max(0, c_hi - c_lo);
#pragma unroll
                    for (int z = 0; z < BK; z++)
                        if ((uint32_t)(z - c_lo - 1) >= seen) x[z] = unseen;
                    if (holes) {
#pragma unroll
                        for (int z = 0; z < BK; z += 16)
                            if (!(head.y >> (z / 16) & 1)) {
#pragma unroll
                                for (int y = 0; y < 16; y++) x[z + y] = unseen;
                            }
                    }
                };
                const bool masked = holes || partial || key0 + BK > len;
                if (masked) mask(-INFINITY);
                float mx4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int z = 4; z < BK; z += 4)
#pragma unroll
                    for (int y = 0; y < 4; y++) mx4[y] = fmaxf(mx4[y], x[z + y]);
                float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), unit_x = fr, shift = 0.0f;
                if constexpr (CAP != kNoCap) {
                    const float cap = a.softcap * 1.44269504f;
                    if constexpr (CAP == kCapCurve) {
                        if (mx > -INFINITY) mx = tanh_of(mx * fr) * cap; /* the curve grows with its argument */
#pragma unroll
                        for (int z = 0; z < BK; z++)
                            if (x[z] != -INFINITY) x[z] = tanh_of(x[z] * fr) * cap;
                        unit_x = 1.0f;
                    } else {
                        /* cap tanh y = cap - 2 cap d, d = 1 / (e^2y + 1): x becomes d, and the rest goes into the weights'
                         * own multiply and add */
                        const float unit = fr * 2.88539008f;
                        if (mx > -INFINITY) mx = fmaf(-2.0f * cap, recip(fl_ex2(mx * unit) + 1.0f), cap);
#pragma unroll
                        for (int z = 0; z < BK; z += 2) {
                            mul2(x[z], x[z + 1], unit, unit);
                            x[z] = fl_ex2(x[z]), x[z + 1] = fl_ex2(x[z + 1]);
                            add2(x[z], x[z + 1], 1.0f, 1.0f);
                            x[z] = recip(x[z]), x[z + 1] = recip(x[z + 1]);
                        }
                        if (masked) mask(INFINITY);
                        unit_x = -2.0f * cap;
                        shift = cap;
                    }
                } else {
                    mx *= fr;
                }
                if (PAIR && j > 0) { /* the other warp's tile moved the reference */
                    if (!(ok = wait_warp(&s_turn[q ^ 1][quarter], (turns + ((j - 1) >> 1)) & 1, abort))) break;
                    const float2 ref = s_ref[row];
                    if (ref.x > m) {
                        l *= fl_ex2(m - ref.x);
                        m = ref.x;
                    }
                    e_acc = (int)ref.y;
                }
                /* O is rescaled when the maximum grew far, or the values' scales did */
                float f = 1.0f;
                bool moved = false;
                if (mx > m + kLazy || (m == -INFINITY && mx > -INFINITY)) {
                    f = fl_ex2(m - mx);
                    l *= f;
                    m = mx;
                    moved = true;
                }
                if (C::ES == 1) {
                    if (head.x > e_acc) {
                        f *= fl_ex2((float)(e_acc - head.x));
                        e_acc = head.x;
                        moved = true;
                    }
                }
                if (PAIR) {
                    s_ref[row] = make_float2(m, (float)e_acc);
                    __syncwarp();
                    if (lane == 0) fl_mbar_arrive(&s_turn[q][quarter]);
                }
                bool odd = false;
                if (partial) {
                    /* what bringing up V found is there once V is */
                    if (!(ok = wait_warp(&v_full[st], (n / ST) & 1, abort))) break;
                    odd = evs[4] | evs[5] | evs[6] | evs[7];
                }
                const bool flush = SPLIT && j > 0 && (j & (C::RUN - 1)) == 0;
                if (flush || (j > 0 && __any_sync(0xffffffffu, moved))) {
                    if (NQ == 1) {
                        /* the products of the tile before are still counted up; for two row tiles S's came after them */
                        if (!(ok = wait_warp(pv_done, (pv_ph + j - 1) & 1, abort))) break;
                        fence_after();
                    }
#pragma unroll 1
                    for (int b = 0; b < HD; b += 32) {
                        float v[32];
                        tmem_ld32(lanes + C::O_COL + mine_q * HD + b, v);
                        tmem_wait_ld(v);
#pragma unroll
                        for (int z = 0; z < 32; z++) v[z] *= f;
                        if (flush) {
                            if (j > C::RUN) add_part(part + b, part_unit(m_part, m, e_part, e_acc), v);
#pragma unroll
                            for (int z = 0; z < 32; z += 4)
                                *reinterpret_cast<float4*>(part + b + z) = make_float4(v[z], v[z + 1], v[z + 2], v[z + 3]);
                        } else {
                            tmem_st32(lanes + C::O_COL + mine_q * HD + b, v);
                        }
                    }
                    if (flush) {
                        m_part = m;
                        e_part = e_acc;
                    } else {
                        tmem_wait_st();
                    }
                }
                if (odd) {
                    /* value elements that are NaN or infinite were left out of the products of a tile that not every
                     * row sees whole: the rows that see them have NaN there in the end */
                    const uint32_t* bits = reinterpret_cast<const uint32_t*>(inf + C::ODD);
                    for (int w = 0; w < HD / 32; w++) {
                        uint32_t b = any_nan ? s_nan[q * 128 + r][w] : 0u;
                        for (int k = max(0, c_lo + 1); k < min(BK, c_hi + 1); k++)
                            if (head.y >> (k >> 4) & 1) b |= bits[k * (HD / 32) + w];
                        s_nan[q * 128 + r][w] = b;
                    }
                    any_nan = true;
                }

                /* weights */
                const float ref = (m == -INFINITY ? 0.0f : m) - (C::ES == 1 ? 0.0f : (float)kUp);
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < BK; b += 32) {
                    uint32_t hi[16], low[16];
#pragma unroll
                    for (int z = b; z < b + 32; z += 4) {
                        fma2(x[z], x[z + 1], unit_x, shift - ref);
                        fma2(x[z + 2], x[z + 3], unit_x, shift - ref);
#pragma unroll
                        for (int y = 0; y < 4; y++) x[z + y] = fl_ex2(x[z + y]);
                        add2(sum[0], sum[1], x[z], x[z + 1]);
                        add2(sum[2], sum[3], x[z + 2], x[z + 3]);
                        if (C::ES == 1) {
                            const float4 v4 = *reinterpret_cast<const float4*>(sv + z);
                            mul2(x[z], x[z + 1], v4.x, v4.y);
                            mul2(x[z + 2], x[z + 3], v4.z, v4.w);
                        }
                        const int i = (z - b) / 2;
                        hi[i] = fl_pack_half2(x[z], x[z + 1]);
                        hi[i + 1] = fl_pack_half2(x[z + 2], x[z + 3]);
                        if (SPLIT) {
                            const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
                            const float2 h1 = __half22float2(*reinterpret_cast<const __half2*>(&hi[i + 1]));
                            low[i] = fl_pack_half2(x[z] - h0.x, x[z + 1] - h0.y);
                            low[i + 1] = fl_pack_half2(x[z + 2] - h1.x, x[z + 3] - h1.y);
                        }
                    }
                    tmem_st16(s_at + b / 2, hi); /* over the scores */
                    if (SPLIT) tmem_st16(lanes + C::LOW_COL + buf * (BK / 2) + b / 2, low);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) fl_mbar_arrive(&p_full[buf]);
            }
            pv_ph += tiles;
            n0 += tiles;
            turns += PAIR ? (tiles + q) >> 1 : 0; /* the other warp's tiles */
            /* ── the output ── */
            if (live) {
                ok = ok && wait_warp(o_full, segs & 1, abort);
                fence_after();
                bool nan_pair[2] = {any_nan, any_nan}; /* of this thread, or of both of the row */
                if constexpr (PAIR) {
                    /* both threads of a row go on with its whole state, and write half of it */
                    s_end[q][row] = make_float4(l, m, any_nan ? 1.0f : 0.0f, m_part);
                    if (q == 0) s_end_e[row] = e_part; /* runs end at even tiles */
                    ok = !pair_any(!ok);
                    const float4 a0 = s_end[0][row], a1 = s_end[1][row];
                    const float2 ref = s_ref[row];
                    m = ref.x;
                    e_acc = (int)ref.y;
                    l = (a0.y == m ? a0.x : a0.x * fl_ex2(a0.y - m)) + (a1.y == m ? a1.x : a1.x * fl_ex2(a1.y - m));
                    m_part = a0.w;
                    e_part = s_end_e[row];
                    nan_pair[0] = a0.z != 0.0f;
                    nan_pair[1] = a1.z != 0.0f;
                    pair_any(false);
                }
                const bool whole = seg.j0 == 0 && seg.j1 == seg.it.tiles;
                const int fold = seg.it.f0 + row, i = fl_div_grp(a, fold), h = seg.head * a.grp + fold - i * a.grp;
                const bool mine = row < seg.it.rows, first = !PAIR || q == 0;
                /* o counts in 2^(e_acc - kUp); F16's weights, and their sum, in 2^-kUp */
                const float unit = fl_scale2(1.0f, (C::ES == 1 ? e_acc : 0) - kUp);
                if (C::ES == 2) l *= 1.0f / (1 << kUp);
                const float inv = whole ? (l == 0.0f ? 0.0f : unit / l) : unit;
                if (mine && first && !whole) ws.ml[slot * RT + row] = make_float2(m, l);
                if (mine && first && whole && a.lse)
                    a.lse[(int64_t)(seg.sw.row0 + i) * a.n_heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.693147181f;
                T* out = static_cast<T*>(a.out) + (int64_t)(seg.sw.row0 + i) * a.out_stride + (int64_t)h * HD;
#pragma unroll
                for (int b0 = 0; b0 < (PAIR ? HD / 2 : HD); b0 += 32) {
                    const int b = PAIR ? q * (HD / 2) + b0 : b0;
                    float v[32];
                    tmem_ld32(lanes + C::O_COL + mine_q * HD + b, v);
                    tmem_wait_ld(v);
                    if (SPLIT && tiles > C::RUN) add_part(part + b, part_unit(m_part, m, e_part, e_acc), v);
                    uint32_t nans = 0;
                    if (PAIR ? nan_pair[0] : nan_pair[q]) nans = s_nan[row][b / 32];
                    if (PAIR && nan_pair[1]) nans |= s_nan[128 + r][b / 32];
#pragma unroll
                    for (int z = 0; z < 32; z += 8) {
                        float x[8];
#pragma unroll
                        for (int y = 0; y < 8; y++) {
                            x[y] = l == 0.0f ? 0.0f : v[z + y] * inv;
                            if (nans >> (z + y) & 1u) x[y] = __uint_as_float(0x7fffffffu);
                        }
                        if (mine && whole) fl_store8(out + b + z, x);
                        if (mine && !whole) fl_store8(part + b + z, x);
                    }
                }
                fence_before();
            }
            segs++;
        }
    }

    fence_before();
    __syncthreads();
    if (warp == kSoftWarps + kLoadWarps) {
        if (lane == 0) /* where a wait ran out the merge kernel makes the rows of this range NaN */
            copy_flag(&static_cast<FlSchedule*>(a.workspace)->expired[blockIdx.x], abort);
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

/* Items that several ranges share, a warp per (row, head). */
template <typename T, int KV, int HD>
__global__ void __launch_bounds__(128) paged_merge_kernel(const FlPaged c, const FlPagedAttn a)
{
    using C = Cfg<KV, HD, sizeof(T) == 4>;
    const int64_t pair = ((int64_t)blockIdx.x * 128 + threadIdx.x) >> 5;
    if (pair >= (int64_t)c.n_rows * a.n_heads) return fl_pdl_wait(); /* this grid may not end before the one it depends on */
    const int row = (int)((uint32_t)pair / (uint32_t)a.n_heads), h = (int)(pair - (int64_t)row * a.n_heads);
    const int seq = fl_row_seq(c.row_start, c.n_seqs, row);
    if (seq < 0) return fl_pdl_wait();
    const SeqWork sw = seq_work<C::RT>(c, a, seq);
    const int head = fl_div_grp(a, h), f = (row - sw.row0) * a.grp + h - head * a.grp, rt = f / C::RT;
    /* units of the head's row tiles, and of those before this one */
    uint32_t all = 0, before = 0;
    for (int x = threadIdx.x & 31; x < sw.nrt; x += 32) {
        const uint32_t u = kItemCost + item_work<C::RT, C::BK>(a, sw, x).tiles;
        all += u;
        before += x < rt ? u : 0;
    }
    all = __reduce_add_sync(0xffffffffu, all);
    before = __reduce_add_sync(0xffffffffu, before);
    const int tiles = item_work<C::RT, C::BK>(a, sw, rt).tiles;
    const FlAttnSpace ws = fl_attn_space(a.workspace, c.n_seqs, kMaxCtas, C::RT, HD);
    fl_pdl_wait();
    const int lane = threadIdx.x & 31;
    const uint32_t* flags = reinterpret_cast<const uint32_t*>(ws.sched->expired);
    const uint32_t any = flags[lane] | (lane < kFlWaitCtas / 4 - 32 ? flags[32 + lane] : 0u);
    const uint32_t per = ws.sched->per;
    const uint32_t t0 = ws.seq_unit[seq] + (uint32_t)head * all + before + kItemCost;
    const int c0 = (int)(t0 / per), c1 = (int)((t0 + tiles - 1) / per);
    if (__any_sync(0xffffffffu, any != 0)) { /* rare: whether one of the item's ranges is meant */
        bool expired = false;
        for (int i = c0 + lane; i <= c1; i += 32) expired |= ws.sched->expired[i] != 0;
        if (__any_sync(0xffffffffu, expired)) return fl_nan_row<T, HD>(a, row, h);
    }
    if (c0 != c1) fl_merge_row<T, HD>(a, ws, c0, c1, f % C::RT, C::RT, row, h); /* else written by its range */
}

template <typename T, int KV, int HD>
cudaError_t launch(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    using C = Cfg<KV, HD, sizeof(T) == 4>;
    static std::atomic<int> sms[64] = {}; /* SMs of a device, once its kernel is configured */
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!sms[dev]) {
        e = cudaFuncSetAttribute(paged_tc_kernel<T, KV, HD, kNoCap>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(paged_tc_kernel<T, KV, HD, kCapCurve>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if constexpr (sizeof(T) == 2)
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(paged_tc_kernel<T, KV, HD, kCapFolded>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        int n = 0;
        e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
        sms[dev] = n < kMaxCtas ? n : kMaxCtas;
    }
    const int grid = sms[dev].load();
    bool folded = false;
    if constexpr (sizeof(T) == 2) {
        folded = a.softcap > 0.0f && a.softcap <= kFoldMax;
        if (folded) paged_tc_kernel<T, KV, HD, kCapFolded><<<grid, kThreads, C::SMEM, st>>>(c, a);
    }
    if (!folded && a.softcap > 0.0f)
        paged_tc_kernel<T, KV, HD, kCapCurve><<<grid, kThreads, C::SMEM, st>>>(c, a);
    else if (!folded)
        paged_tc_kernel<T, KV, HD, kNoCap><<<grid, kThreads, C::SMEM, st>>>(c, a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((int64_t)c.n_rows * a.n_heads + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_merge_kernel<T, KV, HD>, c, a);
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
} // namespace flpt

#endif
