/* fl_paged_tc_hd64.cu — the tcgen05 attention over a paged cache, head_dim 64. */
#include "fl_paged_tc.cuh"

cudaError_t fl_launch_paged_tc_hd64(const FlPaged& c, const FlPagedAttn& a, cudaStream_t st)
{
    return flpt::launch_type<64>(c, a, st);
}
