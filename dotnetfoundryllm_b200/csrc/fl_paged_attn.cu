/*
 * fl_paged_attn.cu — attention of new rows over a paged KV cache
 * (fl_attn_paged_device): workspace, limits and the choice of kernel.
 */
#include "fl_paged_stream.cuh"

using namespace flps;

size_t fl_paged_attn_workspace(const FlPaged& c, int)
{
    size_t bytes;
    workspace(nullptr, c.n_seqs, c.hd, &bytes);
    return bytes;
}

bool fl_paged_attn_fits(const FlPaged& c, int n_heads)
{
    const double items = (double)c.n_rows * n_heads / kRows + (double)c.n_seqs * c.n_kv;
    const double tiles = (double)((int64_t)c.cols << c.page_shift) / kTile;
    return items * (kItemCost + tiles + 1) < 4294967295.0;
}

cudaError_t fl_launch_paged_attn(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    switch (c.hd) {
    case 64: return fl_launch_paged_stream_hd64(c, a, st);
    case 128: return fl_launch_paged_stream_hd128(c, a, st);
    case 256: return fl_launch_paged_stream_hd256(c, a, st);
    default: return cudaErrorInvalidValue;
    }
}
