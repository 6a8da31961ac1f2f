/* fl_paged_hd256.cu — the streaming attention over a paged cache, head_dim 256. */
#include "fl_paged_stream.cuh"

cudaError_t fl_launch_paged_stream_hd256(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    return flps::launch_type<256>(c, a, st);
}
