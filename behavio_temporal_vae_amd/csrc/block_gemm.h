// Matrix products of the gated residual block: bf16 operands (fp32 values as three bf16 planes) or 8-bit e4m3 operands
// with power-of-two block scales, fp32 accumulation on the matrix pipe.
//
//   gemm_rows:  C[m][n] = sum_k A[m][k] B[n][k]      both operands with the reduction contiguous
//   gemm_cols:  C[m][n] = sum_r A[r][m] B[r][n]      both operands with the reduction across rows (weight gradients)
//
// fp32 operands.  A value x is the sum of three bf16 values x0 + x1 + x2 (round to nearest of x, of the rest, of the rest
// of that: |x1| <= 2^-9 |x|, |x2| <= 2^-18 |x|, nothing is lost).  Of the nine products of two such sums the six largest
// are taken; the dropped x1 y2, x2 y1 and x2 y2 are below 2^-26 of x y, four times below an fp32 rounding.  The operands
// arrive as three planes and the kernel runs its reduction over the six plane pairs one after another, smallest first,
// into the same fp32 accumulators: the fp32 form is the bf16 kernel with a reduction six times as long.
//
// Layout of the loop (both kernels).  A workgroup computes a 256 x 256, 128 x 256 or 128 x 128 tile; the reduction goes in stages
// of 64 bytes per row (32 bf16, 64 e4m3), copied global -> LDS without passing through registers into a ring of four
// stages, three of them in flight behind the one being multiplied.  One barrier a stage; the counted waits never drain the
// queue inside the loop.  Pieces of 16 bytes past the end of a row read from a block of zeros instead, so operands need
// no padding beyond a multiple of 8 columns; rows past the end repeat the last row (gemm_rows, where they only reach outputs that
// are not stored) or are zeros (gemm_cols, where rows are the reduction).
#pragma once
#include "common.h"
#include <type_traits>

namespace btvae_block {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int ROWB = 64;                 // bytes of a row in one stage
constexpr int NST = 4;                   // stages in the ring
constexpr int SC_ROW = 128;              // e4m3: scale bytes kept per row of a tile = the reduction blocks one launch may span

enum { FMT_BF16 = 0, FMT_E4M3 = 1 };
enum { EP_LINEAR = 0, EP_GATED = 1, EP_GATED_BWD = 2 };
enum { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2, ACT_SIGMOID = 3 };
enum { T_F32 = 0, T_BF16 = 1, T_PLANES = 2, T_E4M3 = 3 };

struct Args {
    const char* A; long long lda, a_plane;          // byte pitch of rows, bytes between planes
    const char* B; const char* B2; long long ldb, b_plane;      // EP_GATED: B = gate rows, B2 = up rows
    int M, N, K;                                    // N: output columns (EP_GATED: columns of h); K: reduction elements, a multiple of 8
    int pairs;                                      // 1, or 6 plane pairs
    int ks;                                         // stages of one plane pair
    int kz;                                         // stages of one split of the reduction (gridDim.z splits)
    int tiles_m, tiles_n;
    const unsigned char* a_sc; long long a_scp;     // e4m3: scale bytes of A [M][a_scp]
    const unsigned* b_sc; const unsigned* b2_sc; int b_scp;     // e4m3: scale bytes of B's 128-row blocks, four to a word [blocks][b_scp words]
    const void* bias; const void* bias2; int bias_bf16;         // EP_LINEAR: bias; EP_GATED: gate and up
    void* C; long long ldc; int c_type;             // elements; T_F32, T_BF16 (EP_LINEAR), T_PLANES / T_BF16 (one plane) / T_E4M3 / T_F32 (EP_GATED)
    long long c_plane;                              // elements between planes of C
    float* slab;                                    // gridDim.z > 1: fp32 partial results [z][M][N]
    int c_vec;                                      // rows of C start on 16 bytes and columns up to the next multiple of 8 may be written (zeros)
    int act;
    void* gu; long long ldgu; int gu_f32; int gu_half;          // EP_GATED: where a, b are kept (null: not); EP_GATED_BWD: read; b starts gu_half columns after a
    float* colpart;                                 // EP_GATED_BWD: column sums of (da, db) per 64-row strip [strips][2][N], or null
    unsigned char* q_sc; long long q_scp;           // T_E4M3: scale bytes of the output [M][q_scp]
};

__device__ __attribute__((aligned(64))) static const unsigned zero_piece[16] = {0};

__device__ __forceinline__ void glds16(const void* g, void* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}
// Within a wave LDS is served in order: only the compiler has to be kept from moving accesses across.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Byte offset of the logical 16-byte piece c of row r in a stage image of 64-byte rows: the XOR spreads the rows that one
// 16-lane group of a ds_read_b128 touches (the same piece of 16 rows) over all 64 banks.
__device__ __forceinline__ int st_off(int r, int c) { return r * ROWB + ((c ^ ((r >> 2) & 3)) << 4); }

__device__ __forceinline__ unsigned pack2(float a, float b) {
    const f32x2 f = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f, bf16x2));
}
__device__ __forceinline__ float bf_lo(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(unsigned u) { return __uint_as_float(u & 0xFFFF0000u); }
__device__ __forceinline__ float bf_load(const void* p, long long i) { return __uint_as_float((unsigned)reinterpret_cast<const unsigned short*>(p)[i] << 16); }
__device__ __forceinline__ unsigned short bf_bits(float v) { return (unsigned short)(pack2(v, 0.f) & 0xFFFFu); }

// x = p0 + p1 + p2 in bf16.  A finite x whose first rounding would overflow keeps its truncation; a non-finite x is p0 alone.
__device__ __forceinline__ void split3(float x, float& p0, float& p1, float& p2) {
    p0 = bf_lo(pack2(x, 0.f));
    if (!(__builtin_fabsf(p0) < __builtin_inff())) {
        if (__builtin_fabsf(x) < __builtin_inff()) p0 = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
        else { p1 = 0.f; p2 = 0.f; return; }
    }
    const float r = x - p0;
    p1 = bf_lo(pack2(r, 0.f));
    p2 = r - p1;
}

// 8 consecutive values -> 8 bf16 of each plane at element offset o
__device__ __forceinline__ void store_planes8(unsigned short* base, long long plane, int np, long long o, const float (&v)[8]) {
    if (np == 1) {
        u32x4 q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = pack2(v[2 * e], v[2 * e + 1]);
        *reinterpret_cast<u32x4*>(base + o) = q;
        return;
    }
    u32x4 q0, q1, q2;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float a0, a1, a2, b0, b1, b2;
        split3(v[2 * e], a0, a1, a2);
        split3(v[2 * e + 1], b0, b1, b2);
        q0[e] = pack2(a0, b0); q1[e] = pack2(a1, b1); q2[e] = pack2(a2, b2);
    }
    *reinterpret_cast<u32x4*>(base + o) = q0;
    *reinterpret_cast<u32x4*>(base + plane + o) = q1;
    *reinterpret_cast<u32x4*>(base + 2 * plane + o) = q2;
}

// act(a) and act'(a).  FAST (results that are rounded to bf16 or e4m3): the hardware's exp and reciprocal, each good to
// about 2^-22, instead of the correctly rounded division.
template <bool FAST>
__device__ __forceinline__ void act_value(int act, float a, float& v, float& d) {
    if (act == ACT_RELU) { v = a > 0.f ? a : (a == a ? 0.f : a); d = a > 0.f ? 1.f : 0.f; return; }
    if (act == ACT_GELU) {
        const float phi = 0.5f * erfcf(-0.70710678118654752f * a);
        v = a * phi;
        d = phi + a * (FAST ? __expf(-0.5f * a * a) : expf(-0.5f * a * a)) * 0.39894228040143268f;
        return;
    }
    const float s = FAST ? __builtin_amdgcn_rcpf(1.f + __expf(-a)) : 1.f / (1.f + expf(-a));
    if (act == ACT_SILU) { v = a * s; d = s * (1.f + a * (1.f - s)); }
    else { v = s; d = s * (1.f - s); }
}

// Exponent of a block's scale: the smallest e >= -126 with amax <= 448 * 2^e; 0 for a block of zeros.
__device__ __forceinline__ int scale_exp(float amax) {
    if (!(amax > 0.f)) return 0;
    const unsigned u = __float_as_uint(amax);
    const int be = (int)(u >> 23);                                   // biased exponent; a subnormal amax is far below 448 * 2^-126
    const int e = be - 127 - ((u & 0x7FFFFFu) > 0x600000u ? 7 : 8);  // 448 = 1.75 * 2^8
    return e < -126 ? -126 : e;
}
// 2^e for -126 <= e <= 127
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
// four values (already scaled, |v| <= 448) -> four e4m3 bytes, round to nearest even; non-finite values become NaN
__device__ __forceinline__ unsigned pack_e4m3(float a, float b, float c, float d) {
    int r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    return (unsigned)r;
}
__device__ __forceinline__ float finite_abs(float v) {
    const float a = __builtin_fabsf(v);
    return a < __builtin_inff() ? a : 0.f;
}
__device__ __forceinline__ float nan_if_not_finite(float v) { return __builtin_fabsf(v) < __builtin_inff() ? v : __builtin_nanf(""); }

// Tile of this workgroup.  Workgroups are dealt round-robin over the 8 XCDs; each XCD gets a contiguous run of tiles, and
// the run goes through bands of 8 tile rows column by column, so that the 32 tiles an XCD works on at a time share 8 row
// panels and about 4 column panels in its L2.
__device__ __forceinline__ void tile_of(int tiles_m, int tiles_n, int& tm, int& tn) {
    const int T = tiles_m * tiles_n, bid = (int)blockIdx.x;
    const int q = T >> 3, r = T & 7, xcd = bid & 7, idx = bid >> 3;
    const int t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
    const int band = t / (8 * tiles_n), in = t - band * 8 * tiles_n;
    const int rows = min(8, tiles_m - band * 8);
    tm = band * 8 + in % rows;
    tn = in / rows;
}

__device__ __forceinline__ int plane_a(int pair) { return (0x010120 >> (4 * pair)) & 15; }     // pairs (0,2) (2,0) (1,1) (0,1) (1,0) (0,0)
__device__ __forceinline__ int plane_b(int pair) { return (0x001102 >> (4 * pair)) & 15; }

// At most N copies of this wave still in flight, and every LDS read of the stage before done (its slot is about to be refilled).
template <int N> __device__ __forceinline__ void wait_vm() {
    static_assert(N == 0 || N == 4 || N == 6 || N == 8 || N == 12, "");
    if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)" ::: "memory");
    else if constexpr (N == 6) asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
    else if constexpr (N == 8) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(12) lgkmcnt(0)" ::: "memory");
}

// WM x WN waves of 64 x (32 NJ) outputs each.
template <int FMT, int EP, int WM, int WN, int NJ>
__global__ __launch_bounds__(64 * WM * WN, WM * WN == 8 ? 2 : (NJ == 2 ? 2 : 1)) void gemm_rows(const Args p) {
    constexpr int NW = WM * WN, TM = WM * 64, CW = NJ * 32, TN = WN * CW;
    constexpr int STAGE = (TM + TN) * ROWB;
    constexpr int NA = TM / 16 / NW, NB = TN / 16 / NW, NGL = NA + NB;
    constexpr int LDP = CW + 4;                                       // floats per row of a wave's epilogue image
    constexpr int RING = NST * STAGE, EPI_B = NW * 32 * LDP * 4 + (EP == EP_GATED ? TM * WN * 4 : 0);
    constexpr int MAIN = RING > EPI_B ? RING : EPI_B;
    constexpr int SCB = FMT == FMT_E4M3 ? TM * SC_ROW : 0;
    constexpr int SC_AT = RING;                                       // scales sit behind the ring; the epilogue may overwrite them
    __shared__ __attribute__((aligned(1024))) char smem[(RING + SCB > MAIN) ? RING + SCB : MAIN];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wid / WN, wc = wid % WN;
    const int li = lane & 31, lh = lane >> 5;

    int tile_m, tile_n;
    tile_of(p.tiles_m, p.tiles_n, tile_m, tile_n);
    const int m0 = tile_m * TM;
    const int n0 = tile_n * (EP == EP_GATED ? TN / 2 : TN);
    const int zz = (int)blockIdx.z;
    const int s_beg = zz * p.kz, s_end = min(p.pairs * p.ks, s_beg + p.kz);
    const int nk = s_end - s_beg;

    // ---- sources of this wave's copies: instruction j fills 16 rows (1 KiB) of the stage image, a lane one piece of 16 bytes
    const char* asrc[NA];
    const char* bsrc[NB];
    const int piece = (lane & 3) ^ ((lane >> 4) & 3);                 // the logical piece that belongs at this lane's place
#pragma unroll
    for (int j = 0; j < NA; ++j) {
        const int r = (wid * NA + j) * 16 + (lane >> 2);
        asrc[j] = p.A + (long long)min(m0 + r, p.M - 1) * p.lda + (piece << 4);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int r = (wid * NB + j) * 16 + (lane >> 2);
        if constexpr (EP == EP_GATED) {
            // a wave's columns are CW / 2 gate rows followed by the CW / 2 up rows of the same columns of h
            const int c = r / CW, q = r % CW;
            const int f = n0 + c * (CW / 2) + (q % (CW / 2));
            bsrc[j] = (q < CW / 2 ? p.B : p.B2) + (long long)min(f, p.N - 1) * p.ldb + (piece << 4);
        } else {
            bsrc[j] = p.B + (long long)min(n0 + r, p.N - 1) * p.ldb + (piece << 4);
        }
    }
    const bool has_tail = FMT == FMT_BF16 && (p.K & 31) != 0;
    const bool tail_ok = (p.ks - 1) * 32 + piece * 8 < p.K;           // this lane's piece of a last stage lies inside the row
    int pair = s_beg / p.ks, kin = s_beg - pair * p.ks;
    long long aoff = (long long)plane_a(p.pairs == 1 ? 5 : pair) * p.a_plane + (long long)kin * ROWB;
    long long boff = (long long)plane_b(p.pairs == 1 ? 5 : pair) * p.b_plane + (long long)kin * ROWB;
    auto issue = [&](int slot) {
        char* sb = smem + slot * STAGE;
        const bool cut = has_tail && kin == p.ks - 1;                 // uniform
#pragma unroll
        for (int j = 0; j < NA; ++j) {
            const char* s = asrc[j] + aoff;
            if (cut) s = tail_ok ? s : reinterpret_cast<const char*>(zero_piece);
            glds16(s, sb + (wid * NA + j) * 1024);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const char* s = bsrc[j] + boff;
            if (cut) s = tail_ok ? s : reinterpret_cast<const char*>(zero_piece);
            glds16(s, sb + TM * ROWB + (wid * NB + j) * 1024);
        }
        if (++kin == p.ks) {
            kin = 0;
            ++pair;
            aoff = (long long)plane_a(pair) * p.a_plane;
            boff = (long long)plane_b(pair) * p.b_plane;
        } else {
            aoff += ROWB;
            boff += ROWB;
        }
    };

    int oa[2], ob[NJ];
#pragma unroll
    for (int i = 0; i < 2; ++i) oa[i] = st_off(wr * 64 + i * 32 + li, FMT == FMT_BF16 ? lh : 2 * lh);
#pragma unroll
    for (int j = 0; j < NJ; ++j) ob[j] = TM * ROWB + st_off(wc * CW + j * 32 + li, FMT == FMT_BF16 ? lh : 2 * lh);

    f32x16 acc[2][NJ];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // e4m3: the scale bytes of this tile's rows, SC_ROW to a row, over the reduction blocks of this split (whole words of four)
    const unsigned* bs0 = nullptr;
    const unsigned* bs1 = nullptr;
    if constexpr (FMT == FMT_E4M3) {
        const int w0 = s_beg >> 3, nw = (nk + 7) >> 3;                // words of four 128-blocks (eight stages)
        for (int i = tid; i < TM * nw; i += 64 * NW) {
            const int r = i / nw, w = i - r * nw;
            reinterpret_cast<unsigned*>(smem + SC_AT)[r * (SC_ROW / 4) + w] =
                *reinterpret_cast<const unsigned*>(p.a_sc + (long long)min(m0 + r, p.M - 1) * p.a_scp + 4 * (w0 + w));
        }
        if constexpr (EP == EP_GATED) {
            const int blk = (n0 + wc * (CW / 2)) >> 7;                // a wave's columns of h lie in one 128-row block of the weights
            bs0 = p.b_sc + (long long)min(blk, (p.N - 1) >> 7) * p.b_scp + w0;
            bs1 = p.b2_sc + (long long)min(blk, (p.N - 1) >> 7) * p.b_scp + w0;
        } else {
            bs0 = p.b_sc + (long long)min((n0 + wc * CW) >> 7, (p.N - 1) >> 7) * p.b_scp + w0;
        }
        __syncthreads();
    }

#pragma unroll
    for (int s = 0; s < NST - 1; ++s)
        if (s < nk) issue(s);

    int slot = 0, islot = NST - 1;
    unsigned sa4[2] = {0, 0}, sb4[2] = {0, 0};
    for (int t = 0; t < nk; ++t) {
        // stage t has landed once at most the two later stages' copies are in flight
        if (t + 2 < nk) wait_vm<2 * NGL>();
        else if (t + 1 < nk) wait_vm<NGL>();
        else wait_vm<0>();
        __builtin_amdgcn_s_barrier();                                 // everyone's copies of stage t; everyone done with stage t - 1
        __builtin_amdgcn_sched_barrier(0);
        if (t + NST - 1 < nk) issue(islot);                           // into the slot that stage t - 1 left
        const char* sb = smem + slot * STAGE;
        slot = (slot + 1) & (NST - 1);
        islot = (islot + 1) & (NST - 1);
        if constexpr (FMT == FMT_BF16) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                bf16x8 a[2], b[NJ];
#pragma unroll
                for (int i = 0; i < 2; ++i) a[i] = *reinterpret_cast<const bf16x8*>(sb + (oa[i] ^ (s * 32)));
#pragma unroll
                for (int j = 0; j < NJ; ++j) b[j] = *reinterpret_cast<const bf16x8*>(sb + (ob[j] ^ (s * 32)));
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
            }
        } else {
            if ((t & 7) == 0) {                                       // (splits start on a multiple of eight stages)
#pragma unroll
                for (int i = 0; i < 2; ++i) sa4[i] = reinterpret_cast<const unsigned*>(smem + SC_AT)[(wr * 64 + i * 32 + li) * (SC_ROW / 4) + (t >> 3)];
                sb4[0] = bs0[t >> 3];
                if constexpr (EP == EP_GATED) sb4[1] = bs1[t >> 3];
            }
            const int sh = (t & 6) << 2;                              // byte of the word: two stages to a block
            const int sa[2] = {(int)(sa4[0] >> sh), (int)(sa4[1] >> sh)};
            const int sbv[2] = {(int)(sb4[0] >> sh), (int)(sb4[1] >> sh)};
            i32x8 a[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const i32x4 lo = *reinterpret_cast<const i32x4*>(sb + oa[i]), hi = *reinterpret_cast<const i32x4*>(sb + (oa[i] ^ 16));
                a[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const i32x4 lo = *reinterpret_cast<const i32x4*>(sb + ob[j]), hi = *reinterpret_cast<const i32x4*>(sb + (ob[j] ^ 16));
                const i32x8 b = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                const int sbj = (EP == EP_GATED && j >= NJ / 2) ? sbv[1] : sbv[0];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[i], b, acc[i][j], 0, 0, 0, sa[i], 0, sbj);
            }
        }
    }
    __syncthreads();                                                  // all fragments read: the ring becomes the waves' epilogue images

    float* img = reinterpret_cast<float*>(smem) + wid * 32 * LDP;
    float* rowmax = reinterpret_cast<float*>(smem + NW * 32 * LDP * 4);       // [TM][WN] (EP_GATED)
    float cs0[8], cs1[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) cs0[e] = cs1[e] = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        wave_lds_fence();
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) img[((r & 3) + 8 * (r >> 2) + 4 * lh) * LDP + j * 32 + li] = acc[i][j][r];
        wave_lds_fence();
        const int mrow0 = m0 + wr * 64 + i * 32;
        if constexpr (EP == EP_LINEAR) {
            constexpr int LPR = CW / 8, RP = 64 / LPR;                // lanes to a row, rows to a pass
            const int c = (lane % LPR) * 8, n = n0 + wc * CW + c;
            const bool to_slab = gridDim.z > 1;
            float bias[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                bias[e] = (!to_slab && p.bias && n + e < p.N) ? (p.bias_bf16 ? bf_load(p.bias, n + e) : reinterpret_cast<const float*>(p.bias)[n + e]) : 0.f;
#pragma unroll
            for (int pass = 0; pass < 32 / RP; ++pass) {
                const int rr = pass * RP + lane / LPR, m = mrow0 + rr;
                const f32x4 lo = *reinterpret_cast<const f32x4*>(img + rr * LDP + c), hi = *reinterpret_cast<const f32x4*>(img + rr * LDP + c + 4);
                if (m >= p.M || n >= p.N) continue;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = (e < 4 ? lo[e & 3] : hi[e & 3]) + bias[e];
                if (to_slab) {
                    float* d = p.slab + ((long long)zz * p.M + m) * p.N + n;
                    if ((p.N & 3) == 0 && n + 8 <= p.N) {
                        *reinterpret_cast<f32x4*>(d) = f32x4{v[0], v[1], v[2], v[3]};
                        *reinterpret_cast<f32x4*>(d + 4) = f32x4{v[4], v[5], v[6], v[7]};
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) if (n + e < p.N) d[e] = v[e];
                    }
                } else if (p.c_type == T_F32) {
                    float* d = reinterpret_cast<float*>(p.C) + (long long)m * p.ldc + n;
                    if (p.c_vec && n + 8 <= p.N) {
                        *reinterpret_cast<f32x4*>(d) = f32x4{v[0], v[1], v[2], v[3]};
                        *reinterpret_cast<f32x4*>(d + 4) = f32x4{v[4], v[5], v[6], v[7]};
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) if (n + e < p.N) d[e] = v[e];
                    }
                } else {
                    unsigned short* d = reinterpret_cast<unsigned short*>(p.C) + (long long)m * p.ldc + n;
                    if (p.c_vec && n + 8 <= p.N) {
                        *reinterpret_cast<u32x4*>(d) = u32x4{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])};
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) if (n + e < p.N) d[e] = bf_bits(v[e]);
                    }
                }
            }
        } else if constexpr (EP == EP_GATED) {
            constexpr int HW = CW / 2, LPR = HW / 8, RP = 64 / LPR;
            const int c = (lane % LPR) * 8, f = n0 + wc * HW + c;
            float bg[8], bu[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = f + e < p.N;
                bg[e] = (p.bias && in) ? (p.bias_bf16 ? bf_load(p.bias, f + e) : reinterpret_cast<const float*>(p.bias)[f + e]) : 0.f;
                bu[e] = (p.bias2 && in) ? (p.bias_bf16 ? bf_load(p.bias2, f + e) : reinterpret_cast<const float*>(p.bias2)[f + e]) : 0.f;
            }
            const bool quant = p.c_type == T_E4M3;
#pragma unroll
            for (int pass = 0; pass < 32 / RP; ++pass) {
                const int rr = pass * RP + lane / LPR, m = mrow0 + rr;
                float* src = img + rr * LDP + c;
                const f32x4 a0 = *reinterpret_cast<const f32x4*>(src), a1 = *reinterpret_cast<const f32x4*>(src + 4);
                const f32x4 b0 = *reinterpret_cast<const f32x4*>(src + HW), b1 = *reinterpret_cast<const f32x4*>(src + HW + 4);
                float a[8], b[8], h[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    a[e] = (e < 4 ? a0[e & 3] : a1[e & 3]) + bg[e];
                    b[e] = (e < 4 ? b0[e & 3] : b1[e & 3]) + bu[e];
                    float v, d;
                    if (p.c_type == T_BF16 || p.c_type == T_E4M3) act_value<true>(p.act, a[e], v, d);
                    else act_value<false>(p.act, a[e], v, d);
                    h[e] = f + e < p.N ? v * b[e] : 0.f;              // columns between N and the pitch hold zeros
                }
                if (quant) {
                    float mx = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, finite_abs(h[e]));
#pragma unroll
                    for (int o = 1; o < LPR; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
                    if (lane % LPR == 0) rowmax[(wr * 64 + i * 32 + rr) * WN + wc] = mx;
                    *reinterpret_cast<f32x4*>(src) = f32x4{h[0], h[1], h[2], h[3]};       // this lane's own places of the image
                    *reinterpret_cast<f32x4*>(src + 4) = f32x4{h[4], h[5], h[6], h[7]};
                    continue;
                }
                if (m >= p.M || f >= p.N) continue;
                if (p.c_type == T_F32) {
                    float* d = reinterpret_cast<float*>(p.C) + (long long)m * p.ldc + f;  // pitch a multiple of 8
                    *reinterpret_cast<f32x4*>(d) = f32x4{h[0], h[1], h[2], h[3]};
                    *reinterpret_cast<f32x4*>(d + 4) = f32x4{h[4], h[5], h[6], h[7]};
                } else {
                    store_planes8(reinterpret_cast<unsigned short*>(p.C), p.c_plane, p.c_type == T_PLANES ? 3 : 1, (long long)m * p.ldc + f, h);
                }
                if (p.gu) {
                    const long long o = (long long)m * p.ldgu + f;
                    if (p.gu_f32) {
                        float* d = reinterpret_cast<float*>(p.gu) + o;
                        *reinterpret_cast<f32x4*>(d) = f32x4{a[0], a[1], a[2], a[3]};
                        *reinterpret_cast<f32x4*>(d + 4) = f32x4{a[4], a[5], a[6], a[7]};
                        *reinterpret_cast<f32x4*>(d + p.gu_half) = f32x4{b[0], b[1], b[2], b[3]};
                        *reinterpret_cast<f32x4*>(d + p.gu_half + 4) = f32x4{b[4], b[5], b[6], b[7]};
                    } else {
                        unsigned short* d = reinterpret_cast<unsigned short*>(p.gu);
                        store_planes8(d, 0, 1, o, a);
                        store_planes8(d, 0, 1, o + p.gu_half, b);
                    }
                }
            }
            if (quant) {
                __syncthreads();                                      // both column waves' row maxima
#pragma unroll
                for (int pass = 0; pass < 32 / RP; ++pass) {
                    const int rr = pass * RP + lane / LPR, m = mrow0 + rr;
                    const float* src = img + rr * LDP + c;
                    const f32x4 h0 = *reinterpret_cast<const f32x4*>(src), h1 = *reinterpret_cast<const f32x4*>(src + 4);
                    float mx = 0.f;
#pragma unroll
                    for (int w = 0; w < WN; ++w) mx = fmaxf(mx, rowmax[(wr * 64 + i * 32 + rr) * WN + w]);
                    const int e = scale_exp(mx);
                    const float s = pow2i(-e);
                    if (m >= p.M) continue;
                    float h[8];
#pragma unroll
                    for (int q = 0; q < 8; ++q) h[q] = nan_if_not_finite((q < 4 ? h0[q & 3] : h1[q & 3])) * s;
                    // the whole 128-column block is written, zeros beyond N: rows are padded to blocks
                    *reinterpret_cast<u32x2*>(reinterpret_cast<unsigned char*>(p.C) + (long long)m * p.ldc + f) =
                        u32x2{pack_e4m3(h[0], h[1], h[2], h[3]), pack_e4m3(h[4], h[5], h[6], h[7])};
                    if (wc == 0 && lane % LPR == 0) p.q_sc[(long long)m * p.q_scp + tile_n] = (unsigned char)(e + 127);
                }
                __syncthreads();                                      // the images are read before the next 32 rows replace them
            }
        } else {
            constexpr int LPR = CW / 8, RP = 64 / LPR;
            const int c = (lane % LPR) * 8, f = n0 + wc * CW + c;
#pragma unroll
            for (int pass = 0; pass < 32 / RP; ++pass) {
                const int rr = pass * RP + lane / LPR, m = mrow0 + rr;
                const f32x4 lo = *reinterpret_cast<const f32x4*>(img + rr * LDP + c), hi = *reinterpret_cast<const f32x4*>(img + rr * LDP + c + 4);
                if (m >= p.M || f >= p.gu_half) continue;             // zeros from N to gu_half: both halves are one operand of the next product
                float a[8], b[8], da[8], db[8];
                const long long o = (long long)m * p.ldgu + f;
                if (p.gu_f32) {
                    const float* s = reinterpret_cast<const float*>(p.gu) + o;
                    const f32x4 a0 = *reinterpret_cast<const f32x4*>(s), a1 = *reinterpret_cast<const f32x4*>(s + 4);
                    const f32x4 b0 = *reinterpret_cast<const f32x4*>(s + p.gu_half), b1 = *reinterpret_cast<const f32x4*>(s + p.gu_half + 4);
#pragma unroll
                    for (int e = 0; e < 8; ++e) { a[e] = e < 4 ? a0[e & 3] : a1[e & 3]; b[e] = e < 4 ? b0[e & 3] : b1[e & 3]; }
                } else {
                    const unsigned short* s = reinterpret_cast<const unsigned short*>(p.gu) + o;
                    const u32x4 qa = *reinterpret_cast<const u32x4*>(s), qb = *reinterpret_cast<const u32x4*>(s + p.gu_half);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[2 * e] = bf_lo(qa[e]); a[2 * e + 1] = bf_hi(qa[e]);
                        b[2 * e] = bf_lo(qb[e]); b[2 * e + 1] = bf_hi(qb[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float dh = e < 4 ? lo[e & 3] : hi[e & 3];
                    float v, d;
                    if (p.c_type == T_BF16) act_value<true>(p.act, a[e], v, d);
                    else act_value<false>(p.act, a[e], v, d);
                    const bool in = f + e < p.N;
                    da[e] = in ? dh * b[e] * d : 0.f;
                    db[e] = in ? dh * v : 0.f;
                    cs0[e] += da[e];
                    cs1[e] += db[e];
                }
                unsigned short* C = reinterpret_cast<unsigned short*>(p.C);
                const int np = p.c_type == T_PLANES ? 3 : 1;
                store_planes8(C, p.c_plane, np, (long long)m * p.ldc + f, da);
                store_planes8(C, p.c_plane, np, (long long)m * p.ldc + p.gu_half + f, db);
            }
        }
    }
    if constexpr (EP == EP_GATED_BWD) {
        // column sums of this wave's 64 rows, in a fixed order: over a lane's rows above, over the lanes of a column here
        if (p.colpart) {
            constexpr int LPR = CW / 8;
            const int f = n0 + wc * CW + (lane % LPR) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
#pragma unroll
                for (int o = LPR; o < 64; o <<= 1) { cs0[e] += __shfl_xor(cs0[e], o, 64); cs1[e] += __shfl_xor(cs1[e], o, 64); }
            }
            float* d = p.colpart + (long long)(tile_m * WM + wr) * 2 * p.N;
            if (lane < LPR)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (f + e < p.N) { d[f + e] = cs0[e]; d[p.N + f + e] = cs1[e]; }
        }
    }
}

// ---- reduction across rows -----------------------------------------------------------------------------------------
// A stage is 32 rows of both operands, TM / TN columns of 2 bytes.  The MFMA wants eight consecutive reduction steps of one
// column in a lane: two transposing LDS reads (ds_read_b64_tr_b16: a 16-lane group reads 4 rows x 16 columns and lane i gets
// column i) deliver them.  A row of the image is whole multiples of 256 bytes, so rows collide on the banks; the 32-byte granules
// of a row are therefore stored at granule ^ 2 (row & 3), which gives the four rows x two granules that 32 lanes read
// together eight different granules.
struct ColArgs {
    const char* A; long long lda, a_plane; int a_cols;        // byte pitch; columns that may be read (a multiple of 8)
    const char* B; long long ldb, b_plane; int b_cols;
    int R;                                                    // reduction rows
    int M, N;                                                 // outputs
    int pairs, rz;                                            // rows of one split (a multiple of 32)
    int tiles_m, tiles_n;
    float* slab;                                              // [z][M][N]
};

template <int WM, int WN, int NJ>
__global__ __launch_bounds__(64 * WM * WN, WM * WN == 8 ? 2 : (NJ == 2 ? 2 : 1)) void gemm_cols(const ColArgs p) {
    constexpr int NW = WM * WN, TM = WM * 64, CW = NJ * 32, TN = WN * CW;
    constexpr int ARB = TM * 2, BRB = TN * 2;                 // bytes of an image row
    constexpr int STAGE = 32 * (ARB + BRB);
    constexpr int NA = 32 * ARB / 1024 / NW, NB = 32 * BRB / 1024 / NW, NGL = NA + NB;
    constexpr int LDP = CW + 4;
    constexpr int RING = NST * STAGE, EPI_B = NW * 32 * LDP * 4;
    __shared__ __attribute__((aligned(1024))) char smem[RING > EPI_B ? RING : EPI_B];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wid / WN, wc = wid % WN;
    const int li = lane & 31, lh = lane >> 5;
    // Splits of the reduction first: all output tiles of one row range run together on one XCD and share its rows in L2.
    const int T = p.tiles_m * p.tiles_n, nz = (int)gridDim.z;
    int zz, tile;
    if ((nz & 7) == 0) {
        const int L = (int)blockIdx.x + T * (int)blockIdx.z, xcd = L & 7, idx = L >> 3;
        zz = xcd * (nz >> 3) + idx / T;
        tile = idx % T;
    } else {
        zz = (int)blockIdx.z;
        tile = (int)blockIdx.x;
    }
    const int tile_m = tile / p.tiles_n, tile_n = tile % p.tiles_n;
    const int m0 = tile_m * TM, n0 = tile_n * TN;
    const int rbeg = zz * p.rz, rows = max(0, min(p.rz, p.R - rbeg));
    const int ks = (rows + 31) >> 5, nk = ks * p.pairs;

    // instruction j of this wave fills 1 KiB = 1024 / ARB rows of the image
    constexpr int ALR = ARB / 16, BLR = BRB / 16;             // lanes to an image row
    const char* asrc[NA];
    const char* bsrc[NB];
    int arow[NA], brow[NB];
#pragma unroll
    for (int j = 0; j < NA; ++j) {
        const int pos = (wid * NA + j) * 64 + lane, r = pos / ALR, pc = (pos % ALR) ^ ((r & 3) << 2);
        const int col = m0 + pc * 8;
        arow[j] = r;
        asrc[j] = p.A + (long long)(rbeg + r) * p.lda + 2LL * (col + 8 <= p.a_cols ? col : 0);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int pos = (wid * NB + j) * 64 + lane, r = pos / BLR, pc = (pos % BLR) ^ ((r & 3) << 2);
        const int col = n0 + pc * 8;
        brow[j] = r;
        bsrc[j] = p.B + (long long)(rbeg + r) * p.ldb + 2LL * (col + 8 <= p.b_cols ? col : 0);
    }
    int pair = 0, kin = 0;
    long long aoff = (long long)plane_a(p.pairs == 1 ? 5 : 0) * p.a_plane, boff = (long long)plane_b(p.pairs == 1 ? 5 : 0) * p.b_plane;
    auto issue = [&](int slot) {
        char* sb = smem + slot * STAGE;
        const int left = rows - kin * 32;                     // uniform
#pragma unroll
        for (int j = 0; j < NA; ++j) {
            const char* s = asrc[j] + aoff;
            if (left < 32) s = arow[j] < left ? s : reinterpret_cast<const char*>(zero_piece);
            glds16(s, sb + (wid * NA + j) * 1024);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const char* s = bsrc[j] + boff;
            if (left < 32) s = brow[j] < left ? s : reinterpret_cast<const char*>(zero_piece);
            glds16(s, sb + 32 * ARB + (wid * NB + j) * 1024);
        }
        if (++kin == ks) {
            kin = 0;
            ++pair;
            aoff = (long long)plane_a(pair) * p.a_plane;
            boff = (long long)plane_b(pair) * p.b_plane;
        } else {
            aoff += 32 * p.lda;
            boff += 32 * p.ldb;
        }
    };

    // a lane's first transposing read of a 32-column block: row 8 (lane >> 5) + ((lane & 15) >> 2), columns 16 ((lane >> 4) & 1) + 4 (lane & 3)
    const int kr = 8 * lh + ((lane & 15) >> 2), sw = (kr & 3) << 2;
    const int pc0 = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), in8 = (lane & 1) * 8;
    int oa[2], ob[NJ];
#pragma unroll
    for (int i = 0; i < 2; ++i) oa[i] = kr * ARB + ((((wr * 64 + i * 32) / 8 + pc0) ^ sw) << 4) + in8;
#pragma unroll
    for (int j = 0; j < NJ; ++j) ob[j] = 32 * ARB + kr * BRB + ((((wc * CW + j * 32) / 8 + pc0) ^ sw) << 4) + in8;

    f32x16 acc[2][NJ];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    auto frag = [&](const char* q, int rb) {
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)q);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(q + 4 * rb));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };

#pragma unroll
    for (int s = 0; s < NST - 1; ++s)
        if (s < nk) issue(s);
    int slot = 0, islot = NST - 1;
    for (int t = 0; t < nk; ++t) {
        if (t + 2 < nk) wait_vm<2 * NGL>();
        else if (t + 1 < nk) wait_vm<NGL>();
        else wait_vm<0>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (t + NST - 1 < nk) issue(islot);
        const char* sb = smem + slot * STAGE;
        slot = (slot + 1) & (NST - 1);
        islot = (islot + 1) & (NST - 1);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            bf16x8 a[2], b[NJ];
#pragma unroll
            for (int i = 0; i < 2; ++i) a[i] = frag(sb + oa[i] + s * 16 * ARB, ARB);
#pragma unroll
            for (int j = 0; j < NJ; ++j) b[j] = frag(sb + ob[j] + s * 16 * BRB, BRB);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
        }
    }
    __syncthreads();

    float* img = reinterpret_cast<float*>(smem) + wid * 32 * LDP;
    constexpr int LPR = CW / 4, RP = 64 / LPR;                // lanes to a row (4 columns each), rows to a pass
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        wave_lds_fence();
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) img[((r & 3) + 8 * (r >> 2) + 4 * lh) * LDP + j * 32 + li] = acc[i][j][r];
        wave_lds_fence();
        const int c = (lane % LPR) * 4, n = n0 + wc * CW + c;
#pragma unroll
        for (int pass = 0; pass < 32 / RP; ++pass) {
            const int rr = pass * RP + lane / LPR, m = m0 + wr * 64 + i * 32 + rr;
            const f32x4 v = *reinterpret_cast<const f32x4*>(img + rr * LDP + c);
            if (m >= p.M || n >= p.N) continue;
            float* d = p.slab + ((long long)zz * p.M + m) * p.N + n;
            if ((p.N & 3) == 0 && n + 4 <= p.N) *reinterpret_cast<f32x4*>(d) = v;
            else {
#pragma unroll
                for (int e = 0; e < 4; ++e) if (n + e < p.N) d[e] = v[e];
            }
        }
    }
}

}  // namespace btvae_block
