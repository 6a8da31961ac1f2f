/* fl_paged_hd128.cu — the streaming attention over a paged cache, head_dim 128. */
#include "fl_paged_stream.cuh"

cudaError_t fl_launch_paged_stream_hd128(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    return flps::launch_type<128>(c, a, st);
}
