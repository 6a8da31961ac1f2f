/* fl_paged_hd64.cu — the streaming attention over a paged cache, head_dim 64. */
#include "fl_paged_stream.cuh"

cudaError_t fl_launch_paged_stream_hd64(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    return flps::launch_type<64>(c, a, st);
}
