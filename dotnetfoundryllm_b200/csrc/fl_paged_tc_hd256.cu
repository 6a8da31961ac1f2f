/* fl_paged_tc_hd256.cu — the tcgen05 attention over a paged cache, head_dim 256. */
#include "fl_paged_tc.cuh"

cudaError_t fl_launch_paged_tc_hd256(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    return flpt::launch_type<256>(c, a, st);
}
