// Products with the reduction along rows on split (fp32) operands: plain, gated and gated backward results.
#define BTVAE_BLOCK_KERNELS
#include "block_launch.h"

namespace btvae_block {
template int launch_rows<FMT_SPLIT, EP_LINEAR>(Args&, int, hipStream_t, const char*);
template int launch_rows<FMT_SPLIT, EP_GATED_3>(Args&, int, hipStream_t, const char*);
template int launch_rows<FMT_SPLIT, EP_GATED_BWD_3>(Args&, int, hipStream_t, const char*);
}  // namespace btvae_block
