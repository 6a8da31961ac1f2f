/*
 * fl_paged_attn.cu — attention of new rows over a paged KV cache
 * (fl_attn_paged_device): the choice of kernel, workspace and limits.
 */
#include "fl_paged_stream.cuh"
#include "fl_paged_tc.cuh"

namespace {

/* The tcgen05 kernel is taken from this many 16-row tiles per kv head and
 * sequence on (heads of the group included), the streaming one below.  The
 * streaming kernel passes over a sequence's keys once per 16-row tile, so its
 * time is proportional to the tiles; the tcgen05 kernel's is about the same up to
 * 128 rows, but higher for 8 bits (every element is widened into shared memory)
 * and for 32-bit rows (twice the products), which is why the border moves.  It is a
 * rule on the rows of one sequence: a batch goes to one kernel whole, by its longest
 * chunk, and each of its single tokens then takes a row tile of its own (31 tokens
 * beside a chunk of 512 rows, int8: 203 us, as two calls 88 + 44).
 * Measured in us, streaming / tcgen05, 8 kv heads of 4, 16 sequences of 4096 keys
 * (other shapes move the border by how many items share the tcgen05 kernel's start):
 *   rows               16         20         48         64
 *   f16,  F16, 64   43 /  70   66 /  71   91 /  75  115 /  77   from 3 tiles
 *   f16,  F16, 128  71 /  87  120 /  89  175 /  99  229 / 100   from 2
 *   f16,  F16, 256 161 / 134  296 / 134  445 / 142  586 / 144   from 2
 *   f16,  Q8,  64   33 /  83   50 /  84   69 /  86   87 /  89   from 4
 *   bf16, Q8,  128  48 / 118   77 / 119  111 / 128  141 / 129   from 4
 *   bf16, Q8,  256  86 / 159  145 / 160  212 / 165  276 / 166   from 3
 *   bf16, F8,  64   40 /  87   65 /  89   90 /  92  114 /  94   from 3
 *   bf16, F8,  128  74 / 121  125 / 124  178 / 132  230 / 134   from 3
 *   bf16, F8,  256 147 / 168  262 / 169  385 / 173  518 / 175   from 2
 *   f32,  F16, 64   49 / 122   75 / 123  104 / 126  132 / 129   from 4
 *   f32,  F16, 128  91 / 133  156 / 133  229 / 137  305 / 139   from 2
 *   f32,  F16, 256 261 / 270  482 / 270  722 / 277  951 / 280   from 2
 *   f32,  Q8,  64   40 / 149   64 / 150   88 / 152  112 / 154   from 6
 *   f32,  Q8,  128  62 / 166  102 / 166  146 / 169  187 / 170   from 4
 *   f32,  Q8,  256 142 / 300  256 / 300  386 / 307  506 / 309   from 3
 *   f32,  F8,  64   48 / 152   77 / 152  108 / 154  138 / 157   from 5
 *   f32,  F8,  128  90 / 171  151 / 172  220 / 175  281 / 175   from 3
 *   f32,  F8,  256 303 / 307  567 / 307  847 / 315  1116 / 318   from 2 */
int tc_tiles(int kv_dtype, int hd, bool wide)
{
    static constexpr int8_t from[2][3][3] = {{{3, 2, 2}, {4, 4, 3}, {3, 3, 2}}, {{4, 2, 2}, {6, 4, 3}, {5, 3, 2}}};
    return from[wide][kv_dtype - FL_KV_F16][hd == 64 ? 0 : hd == 128 ? 1 : 2];
}

/* The rows of a sequence are the caller's bound, else the average.  `wide`: 32-bit rows. */
bool takes_tc(const FlPaged& c, int n_heads, bool wide)
{
    const int rows = c.max_rows > 0 ? c.max_rows : c.n_seqs > 0 ? (c.n_rows + c.n_seqs - 1) / c.n_seqs : 0;
    return (int64_t)rows * (n_heads / c.n_kv) > flps::kRows * (tc_tiles(c.kv_dtype, c.hd, wide) - 1);
}

} // namespace

/* For every row type: 16-bit rows take the tcgen05 kernel wherever 32-bit ones do, and its space is the larger. */
size_t fl_paged_attn_workspace(const FlPaged& c, int n_heads)
{
    size_t bytes;
    static_assert(flpt::kMaxCtas * 128 >= flps::kMaxCtas * flps::kRows, "the space of either kernel");
    if (takes_tc(c, n_heads, false)) /* row tiles of 256 where two fit, which the bound takes for all types */
        fl_attn_space(nullptr, c.n_seqs, flpt::kMaxCtas, c.hd == 256 ? 128 : 256, c.hd, &bytes);
    else
        fl_attn_space(nullptr, c.n_seqs, flps::kMaxCtas, flps::kRows, c.hd, &bytes);
    return bytes;
}

bool fl_paged_attn_fits(const FlPaged& c, int n_heads)
{
    const bool tc = takes_tc(c, n_heads, true);
    const double rows = tc ? 128 : flps::kRows, keys = tc ? 64 : flps::kTile, start = tc ? flpt::kItemCost : flps::kItemCost;
    const double items = (double)c.n_rows * n_heads / rows + (double)c.n_seqs * c.n_kv;
    return items * (start + (double)((int64_t)c.cols << c.page_shift) / keys + 2) < 4294967295.0;
}

__device__ unsigned int g_expired;

/* Looked up once per device: in a captured call too, which a lookup does not disturb. */
unsigned int* fl_paged_attn_expired(cudaError_t* e)
{
    static std::atomic<unsigned int*> at[64] = {};
    int dev = 0;
    *e = cudaGetDevice(&dev);
    if (*e == cudaSuccess && (dev < 0 || dev >= 64)) *e = cudaErrorInvalidDevice;
    if (*e != cudaSuccess) return nullptr;
    if (!at[dev]) {
        void* p = nullptr;
        *e = cudaGetSymbolAddress(&p, g_expired);
        if (*e != cudaSuccess) return nullptr;
        at[dev] = static_cast<unsigned int*>(p);
    }
    return at[dev];
}

bool fl_paged_attn_waits(const FlPaged& c, int type, int n_heads) { return takes_tc(c, n_heads, type == 0); }

cudaError_t fl_launch_paged_attn(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    const bool tc = takes_tc(c, a.n_heads, a.type == 0);
    switch (c.hd) {
    case 64: return tc ? fl_launch_paged_tc_hd64(c, a, st) : fl_launch_paged_stream_hd64(c, a, st);
    case 128: return tc ? fl_launch_paged_tc_hd128(c, a, st) : fl_launch_paged_stream_hd128(c, a, st);
    case 256: return tc ? fl_launch_paged_tc_hd256(c, a, st) : fl_launch_paged_stream_hd256(c, a, st);
    default: return cudaErrorInvalidValue;
    }
}
