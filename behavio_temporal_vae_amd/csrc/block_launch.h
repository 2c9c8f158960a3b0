// Launches of the products in block_gemm.h.  Their kernels are large: each set is compiled in a file of its own.
#pragma once
#include "block_gemm.h"
#include <algorithm>

namespace btvae_block {

constexpr int CHIP = 256;                                             // compute units
constexpr int MAX_PITCH = 1 << 23;                                    // bytes from row to row of an operand: a tile's rows are found with 32-bit offsets
constexpr int MAX_ROWS = 0x7FE00000;                                  // row numbers, and those a few tiles or splits past them, are 32 bits

inline int tiles(int n, int t) { return (n + t - 1) / t; }
constexpr int tile_width(bool split) { return split ? 128 : 256; }    // columns of gemm_rows' tiles (of 128 rows): see there
inline bool al16(const void* q) { return ((uintptr_t)q & 15) == 0; }

template <int FMT, int EP> int launch_rows(Args& p, int z, hipStream_t s, const char* what);
int launch_cols(const ColPair& p, int split, int big, int z, hipStream_t s);

// Results of more than half the last cache (256 MB, which the operands share) are stored past L2, where they would only drive out the
// operands of other tiles.  Measured, product alone and with a kernel that reads its results, past L2 / through it: e4m3 131,072 x 1000 x 2000 in bf16
// (524 MB) 320 / 369 and 490 / 509 us, 65,536 rows (262 MB) 167 / 177 and 253 / 261, 16,384 rows (66 MB) 47 / 44 and 68 / 66; bf16
// 65,536 x 2000 x 1000 (131 MB) 281 / 331 and 372 / 368; a bf16 unit's forward and backward pass, 1000 -> 2000 -> 1000, its h and their gradients
// past L2 / through it: 65,536 rows (262 and 524 MB) 2714 / 2770, 16,384 rows 790 / 763 us.
constexpr long long STREAM_BYTES = 128ll << 20;

#ifdef BTVAE_BLOCK_KERNELS
// As many workgroups as the chip holds at a time (one of eight waves to a compute unit, or two of four), each going through its items.
template <int FMT, int EP>
int launch_rows(Args& p, int z, hipStream_t s, const char* what) {
    constexpr int WN = tile_width(FMT == FMT_SPLIT) / 64;
    p.tiles_m = tiles(p.M, 128); p.tiles_n = tiles(p.N, 64 * WN / (is_gated(EP) ? 2 : 1)); p.splits = z;
    const long long items = (long long)p.tiles_m * p.tiles_n * z;
    if (p.M > MAX_ROWS) return btvae::set_error("%s: too many rows", what);
    if (items >= (1 << 29)) return btvae::set_error("%s: too many tiles", what);
    if (p.lda >= MAX_PITCH || p.ldb >= MAX_PITCH) return btvae::set_error("%s: rows of more than 8 MiB", what);
    p.stream = z == 1 && (long long)p.M * (EP == EP_GATED_BWD ? 2 * p.half : p.N) * (EP == EP_LINEAR && p.c_type == T_F32 ? 4 : 2) > STREAM_BYTES;
    p.by_tiles = div_by(p.tiles_m * p.tiles_n); p.by_band = div_by(8 * p.tiles_n); p.by_last = div_by(p.tiles_m % 8 ? p.tiles_m % 8 : 8);
    const dim3 grid((unsigned)std::min<long long>(items, FMT == FMT_SPLIT ? 2 * CHIP : CHIP));
    hipLaunchKernelGGL((gemm_rows<FMT, EP, 2, WN, 2, 2>), grid, dim3(128 * WN), 0, s, p);
    return btvae::check_launch(what);
}
#endif

}  // namespace btvae_block
