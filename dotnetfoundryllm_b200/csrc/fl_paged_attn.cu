/*
 * fl_paged_attn.cu — attention of new rows over a paged KV cache
 * (fl_attn_paged_device): the choice of kernel, workspace and limits.
 */
#include "fl_paged_stream.cuh"
#include "fl_paged_tc.cuh"

namespace {

/* Query rows per kv head and sequence, heads of the group included, from which
 * the tcgen05 kernel is taken; below, the streaming one. */
constexpr int kTcRows = 33;

/* The rows of a sequence: the caller's bound, else the average. */
bool takes_tc(const FlPaged& c, int n_heads)
{
    const int rows = c.max_rows > 0 ? c.max_rows : c.n_seqs > 0 ? (c.n_rows + c.n_seqs - 1) / c.n_seqs : 0;
    return (int64_t)rows * (n_heads / c.n_kv) >= kTcRows;
}

} // namespace

size_t fl_paged_attn_workspace(const FlPaged& c, int n_heads)
{
    size_t bytes;
    if (takes_tc(c, n_heads)) /* row tiles of 256 where two fit, which the bound takes for all types */
        fl_attn_space(nullptr, c.n_seqs, flpt::kMaxCtas, c.hd == 256 ? 128 : 256, c.hd, &bytes);
    else
        fl_attn_space(nullptr, c.n_seqs, flps::kMaxCtas, flps::kRows, c.hd, &bytes);
    return bytes;
}

bool fl_paged_attn_fits(const FlPaged& c, int n_heads)
{
    const bool tc = takes_tc(c, n_heads);
    const double rows = tc ? 128 : flps::kRows, keys = tc ? 64 : flps::kTile, start = tc ? flpt::kItemCost : flps::kItemCost;
    const double items = (double)c.n_rows * n_heads / rows + (double)c.n_seqs * c.n_kv;
    return items * (start + (double)((int64_t)c.cols << c.page_shift) / keys + 2) < 4294967295.0;
}

cudaError_t fl_launch_paged_attn(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    const bool tc = takes_tc(c, a.n_heads);
    switch (c.hd) {
    case 64: return tc ? fl_launch_paged_tc_hd64(c, a, st) : fl_launch_paged_stream_hd64(c, a, st);
    case 128: return tc ? fl_launch_paged_tc_hd128(c, a, st) : fl_launch_paged_stream_hd128(c, a, st);
    case 256: return tc ? fl_launch_paged_tc_hd256(c, a, st) : fl_launch_paged_stream_hd256(c, a, st);
    default: return cudaErrorInvalidValue;
    }
}
