// Products with the reduction along rows on e4m3 operands, and those whose results are quantised.
#define BTVAE_BLOCK_KERNELS
#include "block_launch.h"

namespace btvae_block {
template int launch_rows<FMT_E4M3, EP_LINEAR>(Args&, int, hipStream_t, const char*);
template int launch_rows<FMT_E4M3, EP_GATED_Q>(Args&, int, hipStream_t, const char*);
template int launch_rows<FMT_BF16, EP_GATED_Q>(Args&, int, hipStream_t, const char*);
}  // namespace btvae_block
