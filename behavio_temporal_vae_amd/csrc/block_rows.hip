// Products with the reduction along rows, bf16 operands: plain, gated and gated backward results.
#define BTVAE_BLOCK_KERNELS
#include "block_launch.h"

namespace btvae_block {
template int launch_rows<FMT_BF16, EP_LINEAR>(Args&, int, hipStream_t, const char*);
template int launch_rows<FMT_BF16, EP_GATED>(Args&, int, hipStream_t, const char*);
template int launch_rows<FMT_BF16, EP_GATED_BWD>(Args&, int, hipStream_t, const char*);
}  // namespace btvae_block
