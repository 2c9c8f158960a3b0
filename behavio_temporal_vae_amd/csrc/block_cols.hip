// Products with the reduction across rows.
#define BTVAE_BLOCK_KERNELS
#include "block_launch.h"

namespace btvae_block {
int launch_cols(const ColPair& p, int split, int big, int z, hipStream_t s) {
    const dim3 grid((unsigned)p.tiles, 1, (unsigned)z);
    if (split && big) hipLaunchKernelGGL((gemm_cols<true, 2, 2, 4, 4>), grid, dim3(256), 0, s, p);
    else if (split) hipLaunchKernelGGL((gemm_cols<true, 2, 2, 2, 2>), grid, dim3(256), 0, s, p);
    else if (big) hipLaunchKernelGGL((gemm_cols<false, 2, 2, 4, 4>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((gemm_cols<false, 2, 2, 2, 2>), grid, dim3(256), 0, s, p);
    return btvae::check_launch("block_wgrad");
}
}  // namespace btvae_block
