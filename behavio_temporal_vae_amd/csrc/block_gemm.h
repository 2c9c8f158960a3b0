// Matrix products of the gated residual block: bf16 operands (fp32 values as three bf16 planes) or 8-bit e4m3 operands
// with power-of-two block scales, fp32 accumulation on the matrix pipe.
//
//   gemm_rows:  C[m][n] = sum_k A[m][k] B[n][k]      both operands with the reduction contiguous
//   gemm_cols:  C[m][n] = sum_r A[r][m] B[r][n]      both operands with the reduction across rows (weight gradients)
//
// fp32 operands.  A value x is the sum of three bf16 values x0 + x1 + x2 (round to nearest of x, of the rest, of the rest
// of that: |x1| <= 2^-8 |x|, |x2| <= 2^-16 |x|, nothing is lost).  Of the nine products of two such sums the six largest
// are taken; the dropped x1 y2, x2 y1 and x2 y2 are together below 2^-23 of x y and of random sign, about an fp32 rounding.  gemm_rows sums the
// products of first pieces apart from the five small ones, so that a result is rounded once in 16 columns.  A matrix of such
// values ("split") keeps, for every 16 columns, 16 x0, 16 x1 and 16 x2: 96 bytes in a row.  A stage of 16 reduction steps brings
// all three pieces of both operands, so that each piece read from LDS is multiplied twice on average.
//
// gemm_rows.  128 x 256 tiles, eight waves of 64 x 64 and one workgroup to a compute unit (split operands: 128 x 128, four waves, two
// workgroups); the reduction goes in stages of 128 bytes per row (64 bf16, 128 e4m3: whole lines, which is what L2 serves at its full
// rate; split: 96), copied global -> LDS without passing through registers, three stages deep.  A wave reads the operands of its
// next step into a second set of registers while it multiplies the present one; one barrier a stage.  A workgroup goes
// through several tiles: the next tile's stages are on their way while the results of the last one are stored.  Pieces of 16
// bytes past the end of a row read from a block of zeros instead, so operands need no padding beyond a multiple of 8 columns;
// rows past the end repeat the last row and only reach outputs that are not stored.
//   Measured (one card, at 1.7 to 2.0 GHz under these loads; a large library product in bf16 reaches 1394 TFLOP/s):
//   bf16 65,536 x 4000 x 1000 490 to 525 us, 1000 to 1070 TFLOP/s (a library product of this shape 472; operands of zeros, which draw less
//   power, 442 and 404; 128 x 128 tiles of four waves, two stages: 550 us; 256 x 256 tiles of
//   eight waves: 468 us, but their epilogues do not fit the registers); gated 65,536 x 1000 x 2 x 2000 with both projections kept
//   600 to 625 us, 840 to 874 TFLOP/s and 1.03 GB stored; its backward 455 us, 0.8 GB loaded and 0.6 stored; split 16,384 x 4000 x 1000 690 us,
//   190 TFLOP/s of fp32 or 1140 of the products done (a large library product in fp32: 154); e4m3 131,072 x 1000 x 2000
//   320 to 360 us, 1460 to 1640 TFLOP/s; e4m3 gated and quantised again 65,536 x 1000 x 2 x 2000 370 to 440 us, 1190 to 1417 TFLOP/s.
//   What they wait for: the matrix pipe is busy 49 to 66 % of the cycles (epilogues included), the rest are waits at a stage's barrier for operands from L2
//   and LDS; skewing the workgroups against each other, giving waves priorities, or letting a tile's stores pass its successor's first
//   stage changed nothing.
//
// Results.  The weights are the MFMA's first operand, so a lane's 16 results of a 32 x 32 block are 16 columns of ONE row, and the
// weight rows are laid into LDS with bits 2 and 3 of their index swapped, which makes them two runs of 8 consecutive
// columns.  Bias, activation, product and rounding happen there; 2 KiB of LDS to a wave (or 1 KiB twice) then turn each 64 bytes of
// 32 rows over to four neighbouring lanes a row: stores of 16 bytes a lane whose neighbours do not continue them cost several
// times as much (measured: 150 cycles a store instruction instead of about 30).
// A plain product's results leave as whole 128 bytes of a row, through 4 KiB of the slot that is filled next (e4m3 131,072 x 1000 x 2000:
// 366 us instead of 382 with 64 bytes; 240 with nothing stored, 268 of them turned but not stored).  Large ones are stored past L2, which keeps
// the operands of the other tiles there (0.19 GB read beyond L2 instead of 0.47; 329 us): STREAM_BYTES has the rule.
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

constexpr int SC_SLOTS = 4;              // e4m3: groups of four 128-blocks whose scale words are in LDS

enum { FMT_BF16 = 0, FMT_E4M3 = 1, FMT_SPLIT = 2 };
// EP_GATED / EP_GATED_BWD: bf16 operands, results rounded to bf16; EP_GATED_3 / EP_GATED_BWD_3: fp32 values as planes; EP_GATED_Q: h quantised
enum { EP_LINEAR = 0, EP_GATED = 1, EP_GATED_BWD = 2, EP_GATED_3 = 3, EP_GATED_BWD_3 = 4, EP_GATED_Q = 5 };
constexpr bool is_gated(int ep) { return ep == EP_GATED || ep == EP_GATED_3 || ep == EP_GATED_Q; }
enum { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2, ACT_SIGMOID = 3 };
enum { T_F32 = 0, T_BF16 = 1 };

// x / d for 0 <= x < 2^30 by a multiplication: d's reciprocal rounded up to 32 bits behind its leading bit (the error stays below 1 / d)
struct Div {
    unsigned d, mul, shift;
    __host__ __device__ __forceinline__ int of(int x) const {
        return d == 1 ? x : (int)(((unsigned long long)(unsigned)x * mul) >> 32 >> shift);
    }
};
inline Div div_by(int d) {
    Div r = {(unsigned)d, 0u, 0u};
    while ((1u << (r.shift + 1)) < (unsigned)d) ++r.shift;     // 2^shift < d <= 2^(shift + 1)
    if (d > 1) r.mul = (unsigned)(((1ull << (32 + r.shift)) + d - 1) / d);
    return r;
}

constexpr int row_bytes(int fmt) { return fmt == FMT_SPLIT ? 96 : 128; }         // bytes of a row in one stage of gemm_rows

struct Args {
    const char* A; long long lda;                   // byte pitch of rows
    const char* B; const char* B2; long long ldb;   // gated: B = gate rows, B2 = up rows
    int M, N, K;                                    // N: output columns (gated: columns of h); K: reduction elements (bf16: a multiple of 8)
    int ks;                                         // stages of the reduction
    int kz;                                         // stages of one of `splits` splits of it
    int tiles_m, tiles_n, splits;
    Div by_tiles, by_band, by_last;                 // x / tiles, x / (8 tiles_n), x / rows of the last band of 8
    const unsigned char* a_sc; long long a_scp;     // e4m3: scale bytes of A [M][a_scp]
    const unsigned* b_sc; const unsigned* b2_sc; int b_scp;     // e4m3: scale bytes of B's 128-row blocks, four to a word [blocks][b_scp words]
    const void* bias; const void* bias2; int bias_bf16;         // plain: bias; gated: gate and up
    void* C; long long ldc; int c_type;             // EP_LINEAR: T_F32 or T_BF16, pitch in elements; split results: pitch in bytes
    int stream;                                     // bf16 and e4m3 operands: results are stored past L2
    float* slab;                                    // splits > 1: fp32 partial results [z][M][N]
    int act;
    // Gated: where a, b are kept for the backward pass (null: not), in the order in which the kernels' lanes hold them: for every 32 rows and
    // 32 columns a block of a and one of b, 16 values to a lane, each fp32 or (bf16 operands) 24 bits -- 2^-15 instead of bf16's
    // 2^-8, since these values are rounded again as part of the gradients.  Backward: `half` columns of da (a multiple of 32), then db
    char* kept; int half;
    float* colpart;                                 // backward: column sums of (da, db) per wave's strip of rows [strips][2][N], or null
    unsigned char* q_sc; long long q_scp;           // EP_GATED_Q: scale bytes of the output [M][q_scp]
};

__device__ __attribute__((aligned(64))) static const unsigned zero_piece[16] = {0};

__device__ __forceinline__ void glds16(const void* g, void* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}
// The same through a buffer descriptor (a scalar base), at a lane's offset and a scalar one: no address arithmetic, and no wait for every
// LDS read on its way, which the compiler inserts behind the form above.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_at(const void* base) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, -1, 0x00020000); }
__device__ __forceinline__ void blds16(Buffer g, unsigned lane_offset, unsigned offset, void* l) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(g, (__attribute__((address_space(3))) void*)l, 16, lane_offset, offset, 0, 0);
}
// Byte offset of the logical 16-byte piece c of row r in a stage image.  128-byte rows: the XOR spreads the rows that one 16-lane
// group of a ds_read_b128 touches (the same piece of 16 rows) over all 64 banks.  96-byte rows: eight rows do that by
// themselves, the next eight take the other piece of a pair.
template <int FMT> __device__ __forceinline__ int st_swap(int r) { return FMT == FMT_SPLIT ? (r >> 3) & 1 : (r >> 1) & 7; }
template <int FMT> __device__ __forceinline__ int st_off(int r, int c) { return r * row_bytes(FMT) + ((c ^ st_swap<FMT>(r)) << 4); }

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
    const bool finite = __builtin_fabsf(x) < __builtin_inff();
    p0 = bf_lo(pack2(x, 0.f));
    const float cut = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
    p0 = finite && !(__builtin_fabsf(p0) < __builtin_inff()) ? cut : p0;
    const float r = finite ? x - p0 : 0.f;
    p1 = bf_lo(pack2(r, 0.f));
    p2 = r - p1;
}

__device__ __forceinline__ u32x4 pack8(const float (&v)[8]) { return u32x4{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])}; }
__device__ __forceinline__ void split8(const float (&v)[8], u32x4 (&p)[3]) {
    float x[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) split3(v[e], x[0][e], x[1][e], x[2][e]);
#pragma unroll
    for (int k = 0; k < 3; ++k) p[k] = pack8(x[k]);
}
// byte of column c, piece k, in a row of a split matrix
__device__ __forceinline__ long long split_at(int c, int k) { return (long long)(c >> 4) * 96 + k * 32 + (c & 15) * 2; }

typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// act(a) and act'(a).  FAST (results that are rounded to bf16 or e4m3): the hardware's exp and reciprocal, each good to
// about 2^-22, and erfc from Abramowitz and Stegun's 7.1.26 (1.5e-7); otherwise the precise exp and division and erfc from the Chebyshev
// fit t exp(-x^2 + P(t)), t = 1 / (1 + x / 2), of Numerical Recipes (6.2; 1.2e-7 of the value everywhere).
// e^x to about a unit in the last place, for x in [-87, 88] and clamped to it (the product with log2 e in two pieces)
__device__ __forceinline__ float exp_clamped(float x) {
    x = __builtin_amdgcn_fmed3f(x, -87.f, 88.f);
    const float t = x * 1.44269504f, r = __builtin_fmaf(x, 1.92596299e-8f, __builtin_fmaf(x, 1.44269504f, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, r * 0.69314718f, e);
}
// 1 / x for 1 <= x (an infinity as 3e38): the approximate reciprocal and one Newton step.  A result below 2^-126 is 0 (the instruction's, and so the
// step's): the sigmoid below -87.3, whose product with a very negative a is 0 therefore.
__device__ __forceinline__ float reciprocal(float x) {
    x = fminf(x, 3e38f);
    const float y = __builtin_amdgcn_rcpf(x);
    return __builtin_fmaf(__builtin_fmaf(-x, y, 1.f), y, y);
}
// Code of its own for SiLU and GELU (ACT), the others are told apart by `act`: a choice made for every value would cost as much as the value.
template <bool FAST, int ACT>
__device__ __forceinline__ void act_value(int act, float a, float& v, float& d) {
    if constexpr (ACT == ACT_GELU) {
        const float x = __builtin_fabsf(a) * 0.70710678118654752f;
        float g, half_erfc;                                   // exp(-a^2 / 2), erfc(|a| / sqrt 2) / 2
        if constexpr (FAST) {
            const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * x);
            g = __builtin_amdgcn_exp2f(-0.72134752f * a * a);
            half_erfc = 0.5f * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f)))) * g;
        } else {
            const float t = reciprocal(1.f + 0.5f * x);
            const float P = -1.26551223f + t * (1.00002368f + t * (0.37409196f + t * (0.09678418f + t * (-0.18628806f + t * (0.27886807f +
                            t * (-1.13520398f + t * (1.48851587f + t * (-0.82215223f + t * 0.17087277f))))))));
            const float e = -0.5f * a * a;
            g = e < -87.f ? 0.f : exp_clamped(e);             // (a times the clamped value would grow with a)
            half_erfc = 0.5f * t * g * exp_clamped(P);
        }
        const float phi = a < 0.f ? half_erfc : 1.f - half_erfc;
        v = a * phi;
        d = phi + a * g * 0.39894228040143268f;
    } else {
        float s;
        if constexpr (FAST) {
            s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * a));
        } else {
            s = reciprocal(1.f + exp_clamped(-a));
            if constexpr (ACT != ACT_SILU) s = a == a ? s : a;
        }
        if constexpr (ACT == ACT_SILU) {
            v = a * s;
            d = s * (1.f + a * (1.f - s));
        } else {
            v = act == ACT_RELU ? (a > 0.f ? a : (a == a ? 0.f : a)) : s;
            d = act == ACT_RELU ? (a > 0.f ? 1.f : 0.f) : s * (1.f - s);
        }
    }
}
// f(the activation as a constant: SiLU, GELU or -1)
template <class F> __device__ __forceinline__ void with_act(int act, F f) {
    if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>{});
    else if (act == ACT_GELU) f(std::integral_constant<int, ACT_GELU>{});
    else f(std::integral_constant<int, -1>{});
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

// The items (output tiles x splits of the reduction) of this workgroup, one after another.  Workgroups are dealt round-robin over the 8
// XCDs; each XCD gets a contiguous run of items and its workgroups take them in turn.  Tiles run through bands of 8 tile rows
// column by column, so that the 32 an XCD works on at a time share 8 row panels and about 4 column panels in its L2.
struct Items {
    int next, step, end;
    __device__ __forceinline__ explicit Items(int total) {
        const int bid = (int)blockIdx.x, n = (int)gridDim.x, xcd = bid & 7;
        const int q = total >> 3, r = total & 7;
        const int start = xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q;
        next = start + (bid >> 3);
        step = (n - xcd + 7) >> 3;
        end = start + q + (xcd < r);
    }
};
__device__ __forceinline__ void tile_of(const Args& p, int t, int& tm, int& tn) {
    const int band = p.by_band.of(t), in = t - band * 8 * p.tiles_n;
    const bool last = band * 8 + 8 > p.tiles_m;
    const int rows = last ? (int)p.by_last.d : 8;
    tn = last ? p.by_last.of(in) : in >> 3;
    tm = band * 8 + (in - tn * rows);
}

// At most N copies of this wave still in flight, and every LDS read before done (its slot is about to be refilled).  Builtins,
// so that the compiler knows what has been waited for.
template <int N> __device__ __forceinline__ void wait_vm() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));       // vmcnt(N) lgkmcnt(0)
}
__device__ __forceinline__ void meet() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// copies of `per` that belong to step q of `steps`
constexpr int share(int per, int steps, int q) {
    int n = 0;
    for (int j = 0; j < per; ++j) n += j * steps / per == q;
    return n;
}
// Order of a region's instructions: R LDS reads, one behind each of the first matrix instructions (issued in one go they would
// hold the wave up with its matrix pipe idle; issued late their results would), then V copies the same way, of M matrix instructions.
template <int M, int R, int V, int P = 1> __device__ __forceinline__ void spread() {
    constexpr int G = (R + P - 1) / P;
#pragma unroll
    for (int i = 0; i < G; ++i) {
        if (i < M) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, P, 0);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (G + i < M) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
}

// The same with R LDS reads, W LDS writes and V loads, a third of the matrix instructions' worth at a time
template <int M, int R, int V, int W = V> __device__ __forceinline__ void refill() {
    constexpr int ALL = R + V + W;
#pragma unroll
    for (int i = 0; i < M; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
        for (int k = i * ALL / M; k < (i + 1) * ALL / M; ++k) {
            if (k < R) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            else if (k < R + W) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
            else __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        }
    }
}
__device__ __forceinline__ void wait_lds() { wait_vm<63>(); }
// A scalar that the compiler knows nothing about: address and edge computations made from it stay inside their block of results instead of
// being made for all blocks at once and kept, which costs more registers than there are.
__device__ __forceinline__ int opaque(int x) {
    x = __builtin_amdgcn_readfirstlane(x);
    asm volatile("" : "+s"(x));
    return x;
}

// ---- stores and loads of the results' layout ------------------------------------------------------------------------
// A lane's results of one 32-column block: v[q][e] = column 16 q + 8 (lane >> 5) + e of row lane & 31.  `row0`: matrix row of the
// block's row 0, `col0`: matrix column of its column 0.
// HALF: in 1 KiB of LDS to a wave, 16 rows at a time, where the stages leave no more.
template <bool HALF> struct Where {
    static constexpr int LDS_B = HALF ? 1024 : 2048;
    int li, lh, r4, p4, r2, p2;                               // result row and half; row and piece of four / two lanes to a row
    char* lds;
    __device__ __forceinline__ explicit Where(char* wave_lds) : lds(wave_lds) {
        const int lane = threadIdx.x & 63;
        li = lane & 31; lh = lane >> 5; r4 = lane >> 2; p4 = lane & 3; r2 = lane >> 1; p2 = lane & 1;
    }
    // The compiler must not move a lane's reads before other lanes' writes (LDS itself serves a wave in order).
    __device__ __forceinline__ static void fence() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ u32x4* at4(int row, int piece) const { return reinterpret_cast<u32x4*>(lds + row * 64 + ((piece ^ ((row >> 2) & 3)) << 4)); }
    __device__ __forceinline__ char* at2(int row) const { return lds + row * 32; }
    __device__ __forceinline__ static int two(int row) { return ((row >> 3) & 1) << 4; }
    // pieces c0, c1 (16 bytes each) of this lane's row of 64 bytes -> piece p4 of rows r4 and r4 + 16
    __device__ __forceinline__ void turn(const u32x4 x0, int c0, const u32x4 x1, int c1, u32x4& a, u32x4& b) const {
        if constexpr (HALF) {
            if (li < 16) { *at4(li, c0) = x0; *at4(li, c1) = x1; }
            fence();
            a = *at4(r4, p4);
            fence();
            if (li >= 16) { *at4(li - 16, c0) = x0; *at4(li - 16, c1) = x1; }
            fence();
            b = *at4(r4, p4);
        } else {
            *at4(li, c0) = x0;
            *at4(li, c1) = x1;
            fence();
            a = *at4(r4, p4);
            b = *at4(r4 + 16, p4);
        }
        fence();
    }
    // 8-byte pieces lh and 2 + lh of this lane's row of 32 bytes -> 16-byte piece p2 of row r2
    __device__ __forceinline__ u32x4 turn2(const u32x2 x0, const u32x2 x1) const {
        *reinterpret_cast<u32x2*>(at2(li) + ((8 * lh) ^ two(li))) = x0;
        *reinterpret_cast<u32x2*>(at2(li) + ((16 + 8 * lh) ^ two(li))) = x1;
        fence();
        const u32x4 a = *reinterpret_cast<const u32x4*>(at2(r2) + ((16 * p2) ^ two(r2)));
        fence();
        return a;
    }
};
// STREAM: past L2, which holds the operands of other tiles
template <bool STREAM, class T, class V> __device__ __forceinline__ void put_any(T* d, const V v) {
    if constexpr (STREAM) __builtin_nontemporal_store((T)v, d);
    else *d = v;
}
// 8 bf16 (a lane's 16 bytes) at columns c .. c + 7 of a row, those below n only
template <bool STREAM = false> __device__ __forceinline__ void put_bf16(unsigned short* d, const u32x4 v, int c, int n) {
    if (c + 8 <= n) { put_any<STREAM>(reinterpret_cast<u32x4_any*>(d), v); return; }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (c + e < n) d[e] = (unsigned short)(e & 1 ? v[e >> 1] >> 16 : v[e >> 1] & 0xFFFFu);
}
template <bool STREAM = false> __device__ __forceinline__ void put_f32(float* d, const u32x4 u, int c, int n) {
    if (c + 4 <= n) { put_any<STREAM>(reinterpret_cast<f32x4_any*>(d), __builtin_bit_cast(f32x4, u)); return; }
#pragma unroll
    for (int e = 0; e < 4; ++e) if (c + e < n) d[e] = __uint_as_float(u[e]);
}
template <class W> __device__ __forceinline__ void store_bf16(unsigned short* base, long long ld, int row0, int col0, int rows, int cols, const float (&v)[2][8], const W& w) {
    u32x4 a, b;
    w.turn(pack8(v[0]), w.lh, pack8(v[1]), 2 + w.lh, a, b);
    const int c = col0 + 8 * w.p4, r = row0 + w.r4;
    if (c >= cols) return;
    if (r < rows) put_bf16(base + (long long)r * ld + c, a, c, cols);
    if (r + 16 < rows) put_bf16(base + (long long)(r + 16) * ld + c, b, c, cols);
}
__device__ __forceinline__ u32x4 raw4(const float* v) { return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])}; }
template <class W> __device__ __forceinline__ void store_f32(float* base, long long ld, int row0, int col0, int rows, int cols, const float (&v)[2][8], const W& w) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        u32x4 a, b;
        w.turn(raw4(v[q]), 2 * w.lh, raw4(v[q] + 4), 2 * w.lh + 1, a, b);
        const int c = col0 + 16 * q + 4 * w.p4, r = row0 + w.r4;
        if (c >= cols) continue;
        if (r < rows) put_f32(base + (long long)r * ld + c, a, c, cols);
        if (r + 16 < rows) put_f32(base + (long long)(r + 16) * ld + c, b, c, cols);
    }
}
// the block's 192 bytes of each row of a split matrix, 64 at a time (columns are whole groups of 16: `cols` is a multiple of 16)
template <class W> __device__ __forceinline__ void store_split(char* base, long long ld, int row0, int col0, int rows, int cols, const float (&v)[2][8], const W& w) {
    u32x4 p[2][3], a, b;
    split8(v[0], p[0]);
    split8(v[1], p[1]);
    const int r = row0 + w.r4;
#pragma unroll
    for (int t = 0; t < 3; ++t) {                             // bytes 64 t ..: (run 0: pieces 0, 1), (run 0: piece 2, run 1: piece 0), (run 1: pieces 1, 2)
        w.turn(t == 0 ? p[0][0] : (t == 1 ? p[0][2] : p[1][1]), w.lh, t == 0 ? p[0][1] : (t == 1 ? p[1][0] : p[1][2]), 2 + w.lh, a, b);
        const bool in = t == 0 || (t == 1 && w.p4 < 2) || col0 + 16 < cols;
        if (col0 >= cols || !in) continue;
        char* d = base + (long long)r * ld + (long long)(col0 >> 4) * 96 + 64 * t + 16 * w.p4;
        if (r < rows) *reinterpret_cast<u32x4*>(d) = a;
        if (r + 16 < rows) *reinterpret_cast<u32x4*>(d + 16 * ld) = b;
    }
}
// 32 rows of 128 bytes, eight lanes to a row, through 4 KiB of LDS: a row's 16-byte piece `c` of row lane & 31 goes in with `put`, and piece lane & 7 of
// rows 8 k + (lane >> 3) comes out
struct Wide {
    char* lds;
    int li, r8, p8;
    __device__ __forceinline__ explicit Wide(char* wave_lds) : lds(wave_lds) {
        const int lane = threadIdx.x & 63;
        li = lane & 31; r8 = lane >> 3; p8 = lane & 7;
    }
    __device__ __forceinline__ u32x4* at(int row, int piece) const { return reinterpret_cast<u32x4*>(lds + row * 128 + ((piece ^ (row & 7)) << 4)); }
    __device__ __forceinline__ void put(int c, const u32x4 x) const { *at(li, c) = x; }
    __device__ __forceinline__ u32x4 get(int k) const { return *at(8 * k + r8, p8); }
};
// A wave's rows of a matrix of whole 16-byte pieces, through a buffer descriptor that ends behind the last row: pieces outside are not stored.
constexpr unsigned OUTSIDE = 0xFFFFFFF0u;
struct Panel {
    Buffer buf;
    unsigned ld;                                              // bytes
    __device__ __forceinline__ Panel(const void* base, long long ld_bytes, int row0, int rows, int height) : ld((unsigned)ld_bytes) {
        buf = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(reinterpret_cast<const char*>(base)) + row0 * ld_bytes, 0, (unsigned)max(0, min(rows - row0, height)) * (unsigned)ld_bytes, 0x00020000);
    }
    __device__ __forceinline__ unsigned at(int r, unsigned byte, bool in) const { return in ? (unsigned)r * ld + byte : OUTSIDE; }
    __device__ __forceinline__ void put(const u32x4 v, unsigned o, bool stream) const {
        if (stream) __builtin_amdgcn_raw_buffer_store_b128(v, buf, o, 0, 2);       // (uniform; 2: non-temporal)
        else __builtin_amdgcn_raw_buffer_store_b128(v, buf, o, 0, 0);
    }
};
// block of rows `row` .. + 31 of the panel, columns col0 .. + 31 of which those below `cols` (a multiple of 16) exist
template <class W> __device__ __forceinline__ void panel_bf16(const Panel& out, int row, int col0, int cols, const float (&v)[2][8], const W& w, bool stream) {
    u32x4 a, b;
    w.turn(pack8(v[0]), w.lh, pack8(v[1]), 2 + w.lh, a, b);
    const int c = col0 + 8 * w.p4;
    const unsigned o = out.at(row + w.r4, 2 * c, c < cols);
    out.put(a, o, stream);
    out.put(b, c < cols ? o + 16 * out.ld : OUTSIDE, stream);
}
// Kept projections: a block's bytes, and block (row0, col0) of a (0) or b (1); every store and load is 1 KiB in a row
template <bool B24> constexpr int kept_bytes() { return (B24 ? 3 : 4) * 1024; }
template <bool B24> __device__ __forceinline__ char* kept_at(const Args& p, int row0, int col0, int which) {
    return p.kept + (((long long)(row0 >> 5) * (p.half >> 5) + (col0 >> 5)) * 2 + which) * kept_bytes<B24>() + (threadIdx.x & 63) * 16;
}
// Kept projections are next read by the backward pass, long after caches have forgotten them: past L2 both ways (stores past it: a bf16
// forward and backward pass of 4096 / 16,384 / 65,536 rows, 1000 -> 2000 -> 1000, 297 -> 291, 763 -> 747, 2770 -> 2742 us; fp32, 2048 / 16,384 rows: 517 -> 511,
// 3154 -> 3125)
__device__ __forceinline__ void keep_once(char* at, const u32x4 v) { __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(at)); }
struct Raw24 { u32x4 h[2], l; };
struct Raw32 { u32x4 x[4]; };
// 24 bits: the upper three bytes, cut (off by 2^-15 of a value at most, where the gradients made from them are rounded to bf16, 2^-8;
// rounding took four more instructions a value)
__device__ __forceinline__ void keep_24(char* at, const float (&v)[2][8]) {
    u32x4 l;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        unsigned u[8];
        u32x4 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = __float_as_uint(v[q][e]);
#pragma unroll
        for (int d = 0; d < 4; ++d) h[d] = __builtin_amdgcn_perm(u[2 * d + 1], u[2 * d], 0x07060302u);
#pragma unroll
        for (int d = 0; d < 2; ++d)                           // byte 1 of four values
            l[2 * q + d] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[4 * d + 3], u[4 * d + 2], 0x0C0C0501u), __builtin_amdgcn_perm(u[4 * d + 1], u[4 * d], 0x0C0C0501u), 0x05040100u);
        keep_once(at + q * 1024, h);
    }
    keep_once(at + 2048, l);
}
__device__ __forceinline__ u32x4 load_once(const char* at) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at)); }
__device__ __forceinline__ void load_24(const char* at, Raw24& x) {
    x.h[0] = load_once(at);
    x.h[1] = load_once(at + 1024);
    x.l = load_once(at + 2048);
}
__device__ __forceinline__ void unpack_24(const Raw24& x, float (&v)[2][8]) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // bytes 3, 2: the half word, byte 1: the low byte, byte 0: zero
            const unsigned sel = (e & 1 ? 0x07060000u : 0x05040000u) | (unsigned)(e & 3) << 8 | 0x0Cu;
            v[q][e] = __uint_as_float(__builtin_amdgcn_perm(x.h[q][e >> 1], x.l[2 * q + (e >> 2)], sel));
        }
}
__device__ __forceinline__ void keep_32(char* at, const float (&v)[2][8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) keep_once(at + k * 1024, raw4(v[k >> 1] + 4 * (k & 1)));
}
__device__ __forceinline__ void load_32(const char* at, Raw32& x) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x.x[k] = load_once(at + k * 1024);
}
__device__ __forceinline__ void unpack_32(const Raw32& x, float (&v)[2][8]) {
#pragma unroll
    for (int r = 0; r < 16; ++r) v[r >> 3][r & 7] = __uint_as_float(x.x[r >> 2][r & 3]);
}
// Biases are loaded once a tile, before its loop, a column to a lane (a load behind the results' stores would wait for them),
// and read from the lanes: columns c .. c + 31 of what the lanes hold.
__device__ __forceinline__ float bias_lane(const void* bias, int bf16, int col, int cols) {
    if (!bias) return 0.f;                                    // (uniform)
    const int c = min(col, cols - 1);
    return bf16 ? bf_load(bias, c) : reinterpret_cast<const float*>(bias)[c];
}
// (through the wave's LDS: a lane's sixteen values in four reads)
template <class W> __device__ __forceinline__ void put_biases(float lanes, const W& w) {
    reinterpret_cast<float*>(w.lds)[threadIdx.x & 63] = lanes;
    W::fence();
}
template <class W> __device__ __forceinline__ void bias_of(int c, float (&v)[2][8], const W& w) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(w.lds + (c + 16 * q + 8 * w.lh + 4 * k) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][4 * k + e] = x[e];
        }
}
template <class W> __device__ __forceinline__ void clear_beyond(float (&v)[2][8], int col0, int cols, const W& w) {
    if (col0 + 32 <= cols) return;                            // uniform
#pragma unroll
    for (int r = 0; r < 16; ++r)
        if (col0 + 16 * (r >> 3) + 8 * w.lh + (r & 7) >= cols) v[r >> 3][r & 7] = 0.f;
}

// WM x WN waves of (32 MI) x (32 NJ) outputs each
template <int FMT, int EP, int WM, int WN, int MI, int NJ>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_rows(const Args p) {
    constexpr bool GATED = is_gated(EP), FAST = EP != EP_GATED_3 && EP != EP_GATED_BWD_3;
    constexpr bool SPLIT = FMT == FMT_SPLIT;
    constexpr int ROWB = row_bytes(FMT), SLOTS = 3;
    constexpr int NW = WM * WN, RW = MI * 32, CW = NJ * 32, TM = WM * RW, TN = WN * CW;
    constexpr int STAGE = (TM + TN) * ROWB, RING = SLOTS * STAGE;
    constexpr int NA = TM * ROWB / 1024 / NW, NB = TN * ROWB / 1024 / NW;      // copies of a wave and stage
    constexpr int STEPS = FMT == FMT_BF16 ? 4 : 2;            // steps of a stage
    constexpr int SC_B = FMT == FMT_E4M3 ? SC_SLOTS * TM * 4 : 0;
    constexpr int MX_B = EP == EP_GATED_Q ? TM * WN * 4 : 0;  // row maxima of the waves (quantised results)
    typedef Where<FMT == FMT_E4M3 || EP == EP_GATED_Q> Turn;
    __shared__ __attribute__((aligned(1024))) char smem[RING + SC_B + MX_B + NW * Turn::LDS_B];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wid / WN, wc = wid % WN;
    const int li = lane & 31, lh = lane >> 5;
    const Turn wh(smem + RING + SC_B + MX_B + wid * Turn::LDS_B);

    const int T = p.tiles_m * p.tiles_n, all_stages = p.ks;
    const int total_items = T * p.splits;
    Items feed(total_items);                                  // the item being copied: up to two stages ahead of
    Items work = feed;                                        // ... the item being multiplied
    if (feed.next >= feed.end) return;

    // ---- copies: instruction j fills 1 KiB of the stage image (8 rows of 128 bytes, or 10 2/3 of 96: 32 rows to three), a lane one piece of
    // 16 bytes; addresses are a base for the tile and stage (scalar) and a lane's offset from the tile's first row
    constexpr int PR = ROWB / 16;                             // pieces of a row
    auto row_of = [&](int q) { return (q * 64 + lane) / PR; };
    auto piece = [&](int q) { return ((q * 64 + lane) % PR) ^ st_swap<FMT>(row_of(q)); };  // the logical piece that belongs at this lane's place of image part q
    static_assert(!GATED || WM == 2, "");
    const char* const wave_b = GATED && (wid & 1) ? p.B2 : p.B;         // (a wave copies CW / 2 rows, all gate or all up)
    unsigned aofs[NA], bofs[NB];
    const char *abase, *bbase;
    unsigned sofs = 0;
    const unsigned char* scbase = nullptr;
    const bool has_tail = FMT == FMT_BF16 && (p.K & 63) != 0;
    const bool tail_ok[2] = {(p.ks - 1) * 64 + piece(0) * 8 < p.K, (p.ks - 1) * 64 + piece(1) * 8 < p.K};   // this lane's piece of a last stage lies inside the row
    int f_kin = 0, f_left = 0, f_slot = 0, f_scslot = 0;
    long long f_total = 0;                                    // stages still to be copied
    long long koff = 0;
    auto open_feed = [&]() {
        int tm, tn;
        const int zz = p.by_tiles.of(feed.next);
        tile_of(p, feed.next - zz * T, tm, tn);
        const int m0 = tm * TM, n0 = tn * (GATED ? TN / 2 : TN);
        abase = p.A + (long long)m0 * p.lda;
        bbase = wave_b + (long long)n0 * p.ldb;
#pragma unroll
        for (int j = 0; j < NA; ++j)
            aofs[j] = (unsigned)min(row_of(wid * NA + j), p.M - 1 - m0) * (unsigned)p.lda + (piece(wid * NA + j) << 4);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            int r = row_of(wid * NB + j);
            r = (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1);  // bits 2 and 3 swapped: see the results' layout
            if constexpr (GATED) r = (r / CW) * (CW / 2) + r % (CW / 2);       // a wave's columns: CW / 2 gate rows, then the up rows of the same columns of h
            bofs[j] = (unsigned)min(r, p.N - 1 - n0) * (unsigned)p.ldb + (piece(wid * NB + j) << 4);
        }
        const int s_beg = zz * p.kz;
        f_left = min(all_stages, s_beg + p.kz) - s_beg;
        f_kin = s_beg;
        koff = (long long)s_beg * ROWB;
        if constexpr (FMT == FMT_E4M3) {
            scbase = p.a_sc + (long long)m0 * p.a_scp + s_beg;
            sofs = (unsigned)min(tid & (TM - 1), p.M - 1 - m0) * (unsigned)p.a_scp;
        }
    };
    auto next_stage = [&]() {
        if (--f_left == 0) {
            feed.next += feed.step;
            if (feed.next < feed.end) open_feed();
        } else {
            ++f_kin;
            koff += ROWB;
        }
    };
    auto copy_scales = [&]() {
        if constexpr (FMT == FMT_E4M3) {
            if ((f_kin & 3) == 0) {                           // a group of four blocks begins: a scale word of every row (before the stage's own copies)
                if (wid * 64 < TM)
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(scbase + sofs),
                                                     (__attribute__((address_space(3))) void*)(smem + RING + f_scslot * TM * 4 + wid * 256), 4, 0, 0);
                scbase += 4;
                f_scslot = (f_scslot + 1) & (SC_SLOTS - 1);
            }
        }
    };
    auto issue = [&]() {
        char* sb = smem + f_slot * STAGE;
        const char* ab = abase + koff;
        const char* bb = bbase + koff;
        copy_scales();
        if (has_tail && f_kin == p.ks - 1) {                  // uniform
#pragma unroll
            for (int j = 0; j < NA; ++j) glds16(tail_ok[(wid * NA + j) & 1] ? ab + aofs[j] : reinterpret_cast<const char*>(zero_piece), sb + (wid * NA + j) * 1024);
#pragma unroll
            for (int j = 0; j < NB; ++j) glds16(tail_ok[(wid * NB + j) & 1] ? bb + bofs[j] : reinterpret_cast<const char*>(zero_piece), sb + TM * ROWB + (wid * NB + j) * 1024);
        } else {
#pragma unroll
            for (int j = 0; j < NA; ++j) glds16(ab + aofs[j], sb + (wid * NA + j) * 1024);
#pragma unroll
            for (int j = 0; j < NB; ++j) glds16(bb + bofs[j], sb + TM * ROWB + (wid * NB + j) * 1024);
        }
        f_slot = f_slot + 1 == SLOTS ? 0 : f_slot + 1;
        --f_total;
        next_stage();
    };
    {   // stages of all items of this workgroup (only the last split of the reduction is shorter)
        for (int i = feed.next; i < feed.end; i += feed.step) f_total += min(all_stages, (p.by_tiles.of(i) + 1) * p.kz) - p.by_tiles.of(i) * p.kz;
    }
    long long w_total = f_total;                              // stages still to be multiplied

    // operand addresses: piece 2 s + (lane >> 5) of a row at step s (bf16), pieces 4 s + 2 (lane >> 5) and the next (e4m3)
    int oa[MI], ob[NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i) oa[i] = st_off<FMT>(wr * RW + i * 32 + li, FMT == FMT_E4M3 ? 2 * lh : lh);
#pragma unroll
    for (int j = 0; j < NJ; ++j) ob[j] = TM * ROWB + st_off<FMT>(wc * CW + j * 32 + li, FMT == FMT_E4M3 ? 2 * lh : lh);
    typedef typename std::conditional<FMT == FMT_E4M3, i32x8, bf16x8>::type Frag;
    auto frag = [&](const char* sb, int o, int s) -> Frag {
        if constexpr (SPLIT) return *reinterpret_cast<const bf16x8*>(sb + o + s * 32);        // (pairs of pieces: the swap stays within one)
        else if constexpr (FMT == FMT_BF16) return *reinterpret_cast<const bf16x8*>(sb + (o ^ (s * 32)));
        else {
            const i32x4 lo = *reinterpret_cast<const i32x4*>(sb + (o ^ (s * 64))), hi = *reinterpret_cast<const i32x4*>(sb + (o ^ (s * 64) ^ 16));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };
    constexpr int READS = (MI + NJ) * (FMT == FMT_E4M3 ? 2 : 1);          // LDS reads of a step
    // sets of operands: two taken in turn, or (split) the three pieces of A, the three of B and the next stage's first of B
    Frag fa[SPLIT ? 3 : 2][MI], fb[SPLIT ? 4 : 2][NJ];
    f32x16 acc[MI][NJ], low[SPLIT ? MI : 1][SPLIT ? NJ : 1];  // split: sums of the products of first pieces, and of the others
    int sax[MI], sbx[2] = {127, 127};                         // e4m3: the present block's scales
    unsigned sa4[MI], sb4[2] = {0, 0};                        // ... of four blocks
    auto load_set = [&](auto set, const char* sb, int s) {
        constexpr int k = decltype(set)::value & 1;
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[k][i] = frag(sb, oa[i], s);
#pragma unroll
        for (int j = 0; j < NJ; ++j) fb[k][j] = frag(sb, ob[j], s);
    };
    auto product = [&](auto sa, auto sb) {
        constexpr int ka = decltype(sa)::value, k = decltype(sb)::value;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                if constexpr (SPLIT) {
                    f32x16& sum = ka || k ? low[i][j] : acc[i][j];
                    sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[k][j], fa[ka][i], sum, 0, 0, 0);
                } else if constexpr (FMT == FMT_BF16) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[k][j], fa[ka][i], acc[i][j], 0, 0, 0);
                else acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[k][j], fa[ka][i], acc[i][j], 0, 0, 0, (GATED && j >= NJ / 2) ? sbx[1] : sbx[0], 0, sax[i]);
            }
    };
    auto multiply = [&](auto set) { product(std::integral_constant<int, decltype(set)::value & 1>{}, std::integral_constant<int, decltype(set)::value & 1>{}); };
    auto read_a = [&](auto set, const char* sb) {             // split: piece `set` of A, of B (into register set `to`)
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[decltype(set)::value][i] = frag(sb, oa[i], decltype(set)::value);
    };
    auto read_b = [&](auto to, auto set, const char* sb) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) fb[decltype(to)::value][j] = frag(sb, ob[j], decltype(set)::value);
    };
    // the steps of a stage but the last: multiply one, read the next
    // (and, in the steady loop, copies of the stage behind the next, a share to each step)
    constexpr int PER = NA + NB;
    auto copy = [&](auto step, Buffer ab, Buffer bb, unsigned at, char* to) {
        constexpr int q = decltype(step)::value;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j * STEPS / PER == q) {
                if (j < NA) blds16(ab, aofs[j < NA ? j : 0], at, to + (wid * NA + j) * 1024);
                else blds16(bb, bofs[j < NA ? 0 : j - NA], at, to + TM * ROWB + (wid * NB + j - NA) * 1024);
            }
    };
    auto inner = [&](const char* sb, auto copies, Buffer ab, Buffer bb, unsigned at, char* to) {
        constexpr bool C = decltype(copies)::value;
        auto one = [&](auto s) {
            load_set(std::integral_constant<int, decltype(s)::value + 1>{}, sb, decltype(s)::value + 1);
            if constexpr (C) copy(s, ab, bb, at, to);
            multiply(s);
            spread<MI * NJ, READS, C ? share(PER, STEPS, decltype(s)::value) : 0, 2>();
            __builtin_amdgcn_sched_barrier(0);
        };
        one(std::integral_constant<int, 0>{});
        if constexpr (STEPS == 4) {
            one(std::integral_constant<int, 1>{});
            one(std::integral_constant<int, 2>{});
        }
    };
    std::integral_constant<int, 0> S0;
    std::integral_constant<int, 1> S1;                        // (the last step's set: STEPS is even)
    std::integral_constant<int, 2> S2;
    std::integral_constant<int, 3> S3;

    open_feed();
#pragma unroll 1
    for (int s = 0; s < (SPLIT ? 3 : 2); ++s)
        if (f_total > 0) issue();
    if constexpr (SPLIT) f_slot = 0;                          // (also when there were fewer stages than slots)
    int slot = 0, scslot = 0;
    wait_vm<0>();
    meet();
    if constexpr (SPLIT) {
        read_a(S2, smem);
        read_b(S0, S0, smem);
        read_b(S2, S2, smem);
        read_a(S1, smem);
        read_b(S1, S1, smem);
    } else {
        load_set(S0, smem, 0);
    }
    for (; work.next < work.end; work.next += work.step) {
        int tile_m, tile_n;
        const int zz = p.by_tiles.of(work.next);
        tile_of(p, work.next - zz * T, tile_m, tile_n);
        const int m0 = tile_m * TM, n0 = tile_n * (GATED ? TN / 2 : TN);
        const int s_beg = zz * p.kz, nk = min(all_stages, s_beg + p.kz) - s_beg;
        const unsigned* bs0 = nullptr;
        const unsigned* bs1 = nullptr;
        if constexpr (FMT == FMT_E4M3) {                      // (a wave's columns lie in one 128-row block of the weights)
            const int blk = min((n0 + wc * (GATED ? CW / 2 : CW)) >> 7, (p.N - 1) >> 7);
            bs0 = p.b_sc + (long long)blk * p.b_scp + (s_beg >> 2);
            if constexpr (GATED) bs1 = p.b2_sc + (long long)blk * p.b_scp + (s_beg >> 2);
        }
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    acc[i][j][r] = 0.f;
                    if constexpr (SPLIT) low[i][j][r] = 0.f;
                }
        // biases of this wave's columns, a column to a lane: gated, CW / 2 of each, side by side where they fit one register
        float bias_a = 0.f;
        static_assert(CW == 64, "");
        if constexpr (EP == EP_LINEAR) {
            bias_a = bias_lane(p.splits > 1 ? nullptr : p.bias, p.bias_bf16, n0 + wc * CW + lane, p.N);
        } else if constexpr (GATED) {
            const int f = n0 + wc * (CW / 2) + lane % (CW / 2);
            bias_a = bias_lane(p.bias, p.bias_bf16, f, p.N);
            const float up = bias_lane(p.bias2, p.bias_bf16, f, p.N);
            bias_a = lane < 32 ? bias_a : up;
        }
        typedef __attribute__((address_space(4))) unsigned uniform_word;
        auto scales = [&](int t) {                            // a stage is one 128-block
            if constexpr (FMT == FMT_E4M3) {
                if ((t & 3) == 0) {
#pragma unroll
                    for (int i = 0; i < MI; ++i) sa4[i] = reinterpret_cast<const unsigned*>(smem + RING)[scslot * TM + wr * RW + i * 32 + li];
                    sb4[0] = ((const uniform_word*)bs0)[t >> 2];          // (a vector load would wait for every copy on its way)
                    if constexpr (GATED) sb4[1] = ((const uniform_word*)bs1)[t >> 2];
                    scslot = (scslot + 1) & (SC_SLOTS - 1);
                }
                const int sh = (t & 3) << 3;
#pragma unroll
                for (int i = 0; i < MI; ++i) sax[i] = (int)(sa4[i] >> sh);
                sbx[0] = (int)(sb4[0] >> sh);
                sbx[1] = (int)(sb4[1] >> sh);
            }
        };
        // Split operands: products (2,0) (0,2) (1,1) (1,0) (0,1) into one sum, 2^-8 of a result, and (0,0) into another, which so is rounded
        // once in 16 columns and not six times.  A piece's registers take the next stage's piece
        // when its last product has been issued; B's first piece, needed to the end, has a second set.  Behind the first product all
        // of the stage has been read: the waves meet there, and its slot is refilled three stages ahead.
        // Past the last stage the copies go on, of the last rows, into slots that are not read again: one straight path.
        if constexpr (SPLIT) {
            for (int t = 0; t < nk; ++t) {
                const char* cb = smem + slot * STAGE;
                read_a(S0, cb);
                product(S2, S0);
                spread<MI * NJ, MI, 0>();
                __builtin_amdgcn_sched_barrier(0);
                slot = slot + 1 == SLOTS ? 0 : slot + 1;
                wait_vm<NA + NB>();                           // the next stage has landed; the one behind it may be on its way
                meet();
                const char* nb = smem + slot * STAGE;
                char* sb = smem + f_slot * STAGE;
                const Buffer ab = buffer_at(abase), bb = buffer_at(bbase);
                const unsigned at = (unsigned)koff;
                read_a(S2, nb);
                product(S0, S2);
                spread<MI * NJ, MI, 0>();
                __builtin_amdgcn_sched_barrier(0);
                read_b(S3, S0, nb);
                read_b(S2, S2, nb);
                product(S1, S1);
                spread<MI * NJ, 2 * NJ, 0>();
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < NA; ++j) blds16(ab, aofs[j], at, sb + (wid * NA + j) * 1024);
                product(S1, S0);
                spread<MI * NJ, 0, NA>();
                __builtin_amdgcn_sched_barrier(0);
                read_a(S1, nb);
#pragma unroll
                for (int j = 0; j < NB; ++j) blds16(bb, bofs[j], at, sb + TM * ROWB + (wid * NB + j) * 1024);
                product(S0, S1);
                spread<MI * NJ, MI, NB>();
                __builtin_amdgcn_sched_barrier(0);
                read_b(S1, S1, nb);
                product(S0, S0);
                spread<MI * NJ, NJ, 0>();
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < NJ; ++j) fb[0][j] = fb[3][j];
                f_slot = f_slot + 1 == SLOTS ? 0 : f_slot + 1;
                if (f_total > 0) {
                    --f_total;
                    next_stage();
                }
            }
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][j][r] += low[i][j][r];
        }
        if constexpr (!SPLIT) {
            // one stage; the next one's first operands are read behind its last step
            auto stage = [&](int t) {
                if (f_total > 0) issue();                     // into the slot of the stage before
                scales(t);
                inner(smem + slot * STAGE, std::false_type{}, buffer_at(nullptr), buffer_at(nullptr), 0, nullptr);
                slot = slot + 1 == SLOTS ? 0 : slot + 1;
                if (--w_total > 0) {
                    if (w_total - f_total >= 2) wait_vm<PER>();      // the next stage has landed; the one behind it may be on its way
                    else wait_vm<0>();                        // (and earlier results are stored)
                    meet();
                    load_set(S0, smem + slot * STAGE, 0);
                }
                multiply(S1);
            };
            // the same without the cases: the next stage is this tile's, and the copies are whole pieces of the same rows
            auto steady = [&](int t, int run) {
                const Buffer ab = buffer_at(abase), bb = buffer_at(bbase);
                unsigned at = (unsigned)koff;
                for (int left = run; left > 0; --left, ++t) {
                    copy_scales();
                    ++f_kin;
                    scales(t);
                    char* to = smem + f_slot * STAGE;
                    inner(smem + slot * STAGE, std::true_type{}, ab, bb, at, to);
                    slot = slot + 1 == SLOTS ? 0 : slot + 1;
                    f_slot = f_slot + 1 == SLOTS ? 0 : f_slot + 1;
                    wait_vm<PER - share(PER, STEPS, STEPS - 1)>();
                    meet();
                    load_set(S0, smem + slot * STAGE, 0);
                    copy(std::integral_constant<int, STEPS - 1>{}, ab, bb, at, to);
                    at += ROWB;
                    multiply(S1);
                    spread<MI * NJ, READS, share(PER, STEPS, STEPS - 1), 2>();
                    __builtin_amdgcn_sched_barrier(0);
                }
                koff += (long long)run * ROWB;
                f_left -= run; f_total -= run; w_total -= run;
            };
            for (int t = 0; t < nk; ++t) {
                const int run = min(nk - 1 - t, f_left - 1);  // (a last stage may end inside the rows)
                if (f_total > 0 && run > 0) {
                    steady(t, run);
                    t += run;
                }
                stage(t);
            }
        }

        const int row0 = m0 + wr * RW;
        if constexpr (EP == EP_LINEAR) {
            const int col0 = n0 + wc * CW;
            const bool to_slab = p.splits > 1;
            float b[NJ][2][8];
            put_biases(bias_a, wh);
#pragma unroll
            for (int j = 0; j < NJ; ++j) bias_of(j * 32, b[j], wh);
            Turn::fence();
            if constexpr (!SPLIT) {
                // rows of 128 bytes through this wave's part of the slot that is filled next: all waves have read it, and only this wave's copies write there
                static_assert(NB >= 4 && NJ == 2, "");
                const Wide wide(smem + f_slot * STAGE + TM * ROWB + wid * NB * 1024);
                const bool half = !to_slab && p.c_type == T_BF16;
                float* const out = to_slab ? p.slab + (long long)zz * p.M * p.N : reinterpret_cast<float*>(p.C);
                const long long ld = to_slab ? p.N : p.ldc;
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    float v[2][2][8];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int r = 0; r < 16; ++r) v[j][r >> 3][r & 7] = acc[i][j][r] + b[j][r >> 3][r & 7];
                    const int r0 = opaque(row0 + i * 32), c0 = opaque(col0);
                    if (half) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) wide.put(2 * q + lh, pack8(v[q >> 1][q & 1]));
                        Turn::fence();
                        u32x4 x[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[k] = wide.get(k);
                        Turn::fence();
                        const int c = c0 + 8 * wide.p8, r = r0 + wide.r8;
                        if (c < p.N) {
                            unsigned short* d = reinterpret_cast<unsigned short*>(p.C) + (long long)r * p.ldc + c;
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (r + 8 * k < p.M) {
                                    if (p.stream) put_bf16<true>(d + 8 * k * p.ldc, x[k], c, p.N);
                                    else put_bf16(d + 8 * k * p.ldc, x[k], c, p.N);
                                }
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                wide.put(4 * q + 2 * lh, raw4(v[j][q]));
                                wide.put(4 * q + 2 * lh + 1, raw4(v[j][q] + 4));
                            }
                            Turn::fence();
                            u32x4 x[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) x[k] = wide.get(k);
                            Turn::fence();
                            const int c = c0 + 32 * j + 4 * wide.p8, r = r0 + wide.r8;
                            if (c < p.N) {
                                float* d = out + (long long)r * ld + c;
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    if (r + 8 * k < p.M) {
                                        if (p.stream) put_f32<true>(d + 8 * k * ld, x[k], c, p.N);
                                        else put_f32(d + 8 * k * ld, x[k], c, p.N);
                                    }
                            }
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                wait_lds();                                   // (before this wave's copies into the same place)
            } else
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    float v[2][8];
#pragma unroll
                    for (int r = 0; r < 16; ++r) v[r >> 3][r & 7] = acc[i][j][r] + b[j][r >> 3][r & 7];
                    const int r0 = opaque(row0 + i * 32), c0 = opaque(col0 + j * 32);
                    if (to_slab) store_f32(p.slab + (long long)zz * p.M * p.N, p.N, r0, c0, p.M, p.N, v, wh);
                    else if (p.c_type == T_F32) store_f32(reinterpret_cast<float*>(p.C), p.ldc, r0, c0, p.M, p.N, v, wh);
                    else store_bf16(reinterpret_cast<unsigned short*>(p.C), p.ldc, r0, c0, p.M, p.N, v, wh);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        } else if constexpr (GATED) {
            constexpr int HJ = NJ / 2;
            static_assert(HJ == 1, "");
            const Panel out(p.C, 2 * p.ldc, row0, p.M, RW);   // (EP_GATED)
            float bg[2][8], bu[2][8];
            put_biases(bias_a, wh);
            bias_of(0, bg, wh);
            bias_of(32, bu, wh);
            Turn::fence();
            const int col0 = n0 + wc * (CW / 2), N16 = (p.N + 15) & ~15;
            auto gate = [&](auto act) {
#pragma unroll
                for (int j = 0; j < HJ; ++j) {
                    const int c = opaque(col0 + j * 32);
#pragma unroll
                    for (int i = 0; i < MI; ++i) {
                        float a[2][8], b[2][8], h[2][8];
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int q = r >> 3, e = r & 7;
                            a[q][e] = acc[i][j][r] + bg[q][e];
                            b[q][e] = acc[i][j + HJ][r] + bu[q][e];
                            float v, d;
                            act_value<FAST, decltype(act)::value>(p.act, a[q][e], v, d);
                            h[q][e] = v * b[q][e];
                            if (!FAST && (r & 3) == 3) __builtin_amdgcn_sched_barrier(0);
                        }
                        clear_beyond(h, c, p.N, wh);          // columns between N and the pitch hold zeros
                        const int r0 = opaque(row0 + i * 32);
                        if constexpr (EP == EP_GATED_Q) {
#pragma unroll
                            for (int r = 0; r < 16; ++r) acc[i][j][r] = h[r >> 3][r & 7];
                        } else if constexpr (EP == EP_GATED) {
                            panel_bf16(out, i * 32, c, N16, h, wh, p.stream);
                            if (p.kept && r0 < p.M && c < p.half) {         // (uniform)
                                keep_24(kept_at<true>(p, r0, c, 0), a);
                                keep_24(kept_at<true>(p, r0, c, 1), b);
                            }
                        } else {
                            if (p.kept && r0 < p.M && c < p.half) {         // (uniform)
                                keep_32(kept_at<false>(p, r0, c, 0), a);
                                keep_32(kept_at<false>(p, r0, c, 1), b);
                            }
                            __builtin_amdgcn_sched_barrier(0);
                            store_split(reinterpret_cast<char*>(p.C), p.ldc, r0, c, p.M, N16, h, wh);
                        }
                        __builtin_amdgcn_sched_barrier(0);    // one block at a time: mixing them costs more registers than there are
                    }
                }
            };
            with_act(p.act, gate);
            if constexpr (EP == EP_GATED_Q) {                 // the tile's 128 columns of h are one block of every row
                static_assert(WN * CW == 256, "");
                float* mx = reinterpret_cast<float*>(smem + RING + SC_B);
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    float m = 0.f;
#pragma unroll
                    for (int j = 0; j < HJ; ++j)
#pragma unroll
                        for (int r = 0; r < 16; ++r) m = fmaxf(m, finite_abs(acc[i][j][r]));
                    m = fmaxf(m, __shfl_xor(m, 32, 64));
                    if (lh == 0) mx[(wr * RW + i * 32 + li) * WN + wc] = m;
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    float m = 0.f;
#pragma unroll
                    for (int w = 0; w < WN; ++w) m = fmaxf(m, mx[(wr * RW + i * 32 + li) * WN + w]);
                    const int r0 = opaque(row0 + i * 32), e = scale_exp(m), row = r0 + li;
                    const float s = pow2i(-e);
                    if (wc == 0 && lh == 0 && row < p.M) p.q_sc[(long long)row * p.q_scp + tile_n] = (unsigned char)(e + 127);
#pragma unroll
                    for (int j = 0; j < HJ; ++j) {
                        unsigned u[2][2];
#pragma unroll
                        for (int r = 0; r < 16; r += 4)
                            u[r >> 3][(r >> 2) & 1] = pack_e4m3(nan_if_not_finite(acc[i][j][r]) * s, nan_if_not_finite(acc[i][j][r + 1]) * s,
                                                                nan_if_not_finite(acc[i][j][r + 2]) * s, nan_if_not_finite(acc[i][j][r + 3]) * s);
                        // the whole 128-column block is written, zeros beyond N: rows are padded to blocks
                        const u32x4 x = wh.turn2(u32x2{u[0][0], u[0][1]}, u32x2{u[1][0], u[1][1]});
                        const int c = opaque(col0 + j * 32) + 16 * wh.p2, r = r0 + wh.r2;
                        if (r < p.M) *reinterpret_cast<u32x4*>(reinterpret_cast<unsigned char*>(p.C) + (long long)r * p.ldc + c) = x;
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                __syncthreads();                              // the maxima are read before the next tile's replace them
            }
        } else {
            const int col0 = n0 + wc * CW, strip = tile_m * WM + wr;
            const Panel out_a(p.C, 2 * p.ldc, row0, p.M, RW), out_b(reinterpret_cast<unsigned short*>(p.C) + p.half,      // (FAST)
                        2 * p.ldc, row0, p.M, RW);
            auto gate = [&](auto act) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int c = opaque(col0 + j * 32);
                    if (c >= p.half) continue;             // (uniform)
                    float cs[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) cs[k] = 0.f;
                    auto one = [&](int i, float (&a)[2][8], float (&b)[2][8]) {
                        float da[2][8], db[2][8];
                        const int r0 = opaque(row0 + i * 32);
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int q = r >> 3, e = r & 7;
                            float v, d;
                            act_value<FAST, decltype(act)::value>(p.act, a[q][e], v, d);
                            const float dh = acc[i][j][r];
                            da[q][e] = dh * b[q][e] * d;
                            db[q][e] = dh * v;
                            if (!FAST && (r & 3) == 3) __builtin_amdgcn_sched_barrier(0);
                        }
                        if (r0 + 32 > p.M && r0 + li >= p.M) {      // (rows behind the last take no part in the sums)
#pragma unroll
                            for (int r = 0; r < 16; ++r) da[r >> 3][r & 7] = db[r >> 3][r & 7] = 0.f;
                        }
                        clear_beyond(da, c, p.N, wh);         // zeros from N to half: both halves are one operand of the next product
                        clear_beyond(db, c, p.N, wh);
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            cs[r] += da[r >> 3][r & 7];
                            cs[16 + r] += db[r >> 3][r & 7];
                        }
                        if constexpr (FAST) {
                            panel_bf16(out_a, i * 32, c, p.half, da, wh, p.stream);
                            panel_bf16(out_b, i * 32, c, p.half, db, wh, p.stream);
                        } else {
                            store_split(reinterpret_cast<char*>(p.C), p.ldc, r0, c, p.M, p.half, da, wh);
                            store_split(reinterpret_cast<char*>(p.C) + split_at(p.half, 0), p.ldc, r0, c, p.M, p.half, db, wh);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    };
                    if constexpr (FAST) {
                        Raw24 ra[MI], rb[MI];
#pragma unroll
                        for (int i = 0; i < MI; ++i) {
                            const int rl = min(opaque(row0 + i * 32), (p.M - 1) & ~31);      // (a block that exists)
                            load_24(kept_at<true>(p, rl, c, 0), ra[i]);
                            load_24(kept_at<true>(p, rl, c, 1), rb[i]);
                        }
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int i = 0; i < MI; ++i) {
                            float a[2][8], b[2][8];
                            unpack_24(ra[i], a);
                            unpack_24(rb[i], b);
                            one(i, a, b);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < MI; ++i) {
                            float a[2][8], b[2][8];
                            Raw32 ra, rb;
                            const int rl = min(opaque(row0 + i * 32), (p.M - 1) & ~31);
                            load_32(kept_at<false>(p, rl, c, 0), ra);
                            load_32(kept_at<false>(p, rl, c, 1), rb);
                            unpack_32(ra, a);
                            unpack_32(rb, b);
                            one(i, a, b);
                        }
                    }
                    if (p.colpart) {
                        // sums over the 32 rows of a half wave, in a fixed order, halving the values a lane holds with every step: lane
                        // (li, lh) ends with the sum of value li
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) {
                            const bool hi = (lane & o) != 0;
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                if (k < o) {
                                    const float keep = hi ? cs[k + o] : cs[k], give = hi ? cs[k] : cs[k + o];
                                    cs[k] = keep + __shfl_xor(give, o, 64);
                                }
                        }
                        const int r = li & 15, col = c + 16 * (r >> 3) + 8 * lh + (r & 7);
                        if (col < p.N) p.colpart[((long long)strip * 2 + (li >> 4)) * p.N + col] = cs[0];
                    }
                }
            };
            with_act(p.act, gate);
        }
    }
    if constexpr (SPLIT) wait_vm<0>();                        // no copy may still be on its way when the LDS passes to others
}

// ---- reduction across rows -----------------------------------------------------------------------------------------
// A stage is 32 rows of both operands, TM / TN columns of 2 bytes (split operands: 16 rows, 6 bytes a column).  The MFMA wants
// eight consecutive reduction steps of one column in a lane: two transposing LDS reads (ds_read_b64_tr_b16: a 16-lane group
// reads 4 rows x 16 columns and lane i gets column i) deliver them.  A row of the image is whole multiples of 256 bytes, so
// rows collide on the banks; the 32-byte granules of a row are therefore stored at granule ^ 2 (row & 3), which gives the four
// rows x two granules (neighbours, or three apart in a split row) that 32 lanes read together eight different places.
// Stages come through registers, two ahead (split: one), and are written to one of three LDS slots: the compiler waits for every copy
// global -> LDS on its way before a transposing read, so that such copies would not overlap anything (768 us instead of 545 below).
// Four waves, 256 x 256 tiles of one workgroup a compute unit where the splits of the rows fill the chip with them, else 128 x 128 and two.
//   Measured, 256 / 128 tiles: bf16 65,536 rows, 4032 x 1000: 546 / 707 us (968 TFLOP/s; a library product of the shape 687), 16,384 rows
//   1000 x 2000 86 / 94 us, 4096 rows 44 / 37 us, 65,536 rows 512 x 256 63 / 45 us; split 16,384 rows, 4032 x 1000: 608 / 717 us (217
//   TFLOP/s of fp32, 1300 of the products done), 2048 rows 1024 x 1024 50 / 38 us.  What bounds it: transposing reads (as many LDS
//   cycles as matrix cycles) behind one wave to a SIMD; the matrix pipe is busy 52 % of the cycles, split 73 %.
struct ColArgs {
    const char* A; long long lda; int a_cols;                 // byte pitch; columns that may be read (a multiple of 8; split: of 16)
    const char* B; long long ldb; int b_cols;
    int R;                                                    // reduction rows
    int M, N;                                                 // outputs
    int rz;                                                   // rows of one split (a multiple of 32)
    int tiles_m, tiles_n;
    float* slab;                                              // [z][M][N]
};
// One product, or two over the same rows and splits side by side (small ones do not fill the chip, and a launch less is most of their time)
struct ColPair { ColArgs a[2]; int tiles0, tiles; };          // tiles of the first, of both


template <bool SPLIT, int WM, int WN, int MI, int NJ>
__global__ __launch_bounds__(64 * WM * WN, MI * NJ == 16 ? 1 : 2) void gemm_cols(const ColPair pair) {
    constexpr int NW = WM * WN, RW = MI * 32, CW = NJ * 32, TM = WM * RW, TN = WN * CW;
    constexpr int EB = SPLIT ? 6 : 2, SR = SPLIT ? 16 : 32, SLOTS = 3, SETS = SPLIT ? 1 : 2;        // bytes of a column, rows of a stage, stages in LDS and in registers
    constexpr int ARB = TM * EB, BRB = TN * EB;               // bytes of an image row
    constexpr int STAGE = SR * (ARB + BRB), RING = SLOTS * STAGE;
    constexpr int NA = SR * ARB / 1024 / NW, NB = SR * BRB / 1024 / NW, NGL = NA + NB;
    __shared__ __attribute__((aligned(1024))) char smem[RING + NW * Where<false>::LDS_B];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wid / WN, wc = wid % WN;
    const int lh = lane >> 5;
    const Where<false> wh(smem + RING + wid * Where<false>::LDS_B);
    // Each XCD (every eighth workgroup) gets a contiguous run of the tiles of one row range after another: neighbouring tiles share that range's
    // rows in its L2 (measured, 65,536 rows of 4032 x 1000 in four ranges: 2.4 -> 0.8 GB read beyond it, 585 -> 575 us)
    const int T = pair.tiles, total = T * (int)gridDim.z, L = (int)blockIdx.x + T * (int)blockIdx.z, xcd = L & 7, q = total >> 3, rem = total & 7;
    const int item = (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + (L >> 3);
    const int zz = item / T;
    int tile = item % T;
    const ColArgs& p = pair.a[tile >= pair.tiles0];
    if (tile >= pair.tiles0) tile -= pair.tiles0;
    const int tile_m = tile / p.tiles_n, tile_n = tile % p.tiles_n;
    const int m0 = tile_m * TM, n0 = tile_n * TN;
    const int rbeg = zz * p.rz, rows = max(0, min(p.rz, p.R - rbeg));
    const int nk = (rows + SR - 1) / SR;

    // instruction j of this wave fills 1 KiB of the image; a piece of 16 bytes past the readable columns reads the row's first instead
    constexpr int ALR = ARB / 16, BLR = BRB / 16;             // pieces of an image row
    unsigned aofs[NA], bofs[NB];
    int arow[NA], brow[NB];
    auto column = [&](int c0, int pc, int cols) -> unsigned {
        if constexpr (SPLIT) return c0 + (pc / 6) * 16 < cols ? (unsigned)(c0 / 16 * 96 + pc * 16) : 0u;
        else return c0 + pc * 8 < cols ? 2u * (unsigned)(c0 + pc * 8) : 0u;
    };
#pragma unroll
    for (int j = 0; j < NA; ++j) {
        const int pos = (wid * NA + j) * 64 + lane, r = pos / ALR;
        arow[j] = r;
        aofs[j] = (unsigned)r * (unsigned)p.lda + column(m0, (pos % ALR) ^ ((r & 3) << 2), p.a_cols);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int pos = (wid * NB + j) * 64 + lane, r = pos / BLR;
        brow[j] = r;
        bofs[j] = (unsigned)r * (unsigned)p.ldb + column(n0, (pos % BLR) ^ ((r & 3) << 2), p.b_cols);
    }
    const char* ab = p.A + (long long)rbeg * p.lda;
    const char* bb = p.B + (long long)rbeg * p.ldb;
    const char* zero = reinterpret_cast<const char*>(zero_piece);
    int f_slot = 0, left = rows;                              // rows not yet loaded
    typedef __attribute__((address_space(1))) u32x4 global_u32x4;
    u32x4 regs[SETS][NGL];
    // One stage's loads; rows past the end are zeros, and past the last stage all of them are: one straight path
    auto fetch_a = [&](auto set) {
#pragma unroll
        for (int j = 0; j < NA; ++j) regs[decltype(set)::value][j] = *(const global_u32x4*)(arow[j] < left ? ab + aofs[j] : zero);
    };
    auto fetch_b = [&](auto set) {
#pragma unroll
        for (int j = 0; j < NB; ++j) regs[decltype(set)::value][NA + j] = *(const global_u32x4*)(brow[j] < left ? bb + bofs[j] : zero);
        ab += SR * p.lda;
        bb += SR * p.ldb;
        left -= SR;
    };
    auto put_a = [&](auto set) {
#pragma unroll
        for (int j = 0; j < NA; ++j) *reinterpret_cast<u32x4*>(smem + f_slot * STAGE + (wid * NA + j) * 1024 + lane * 16) = regs[decltype(set)::value][j];
    };
    auto put_b = [&](auto set) {
#pragma unroll
        for (int j = 0; j < NB; ++j) *reinterpret_cast<u32x4*>(smem + f_slot * STAGE + SR * ARB + (wid * NB + j) * 1024 + lane * 16) = regs[decltype(set)::value][NA + j];
        f_slot = f_slot + 1 == SLOTS ? 0 : f_slot + 1;
    };

    // a lane's first transposing read of a 32-column block: row 8 (lane >> 5) + ((lane & 15) >> 2), columns 16 ((lane >> 4) & 1) + 4 (lane & 3)
    constexpr int PC = SPLIT ? 3 : 1;                         // pieces of a value
    const int kr = 8 * lh + ((lane & 15) >> 2);
    auto granule = [&](int c, int k) { return ((((c >> 4) + ((lane >> 4) & 1)) * PC + k) ^ ((kr & 3) << 1)) * 32 + (lane & 3) * 8; };
    int oa[PC][MI], ob[PC][NJ];
#pragma unroll
    for (int k = 0; k < PC; ++k) {
#pragma unroll
        for (int i = 0; i < MI; ++i) oa[k][i] = kr * ARB + granule(wr * RW + i * 32, k);
#pragma unroll
        for (int j = 0; j < NJ; ++j) ob[k][j] = SR * ARB + kr * BRB + granule(wc * CW + j * 32, k);
    }

    f32x16 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
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
    bf16x8 fa[SPLIT ? 3 : 2][MI], fb[SPLIT ? 4 : 2][NJ];
    // register set `to` of A / B: piece k (split), or step s of 16 rows
    auto read_a = [&](auto to, int k, const char* sb, int s) {
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[decltype(to)::value][i] = frag(sb + oa[k][i] + s * 16 * ARB, ARB);
    };
    auto read_b = [&](auto to, int k, const char* sb, int s) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) fb[decltype(to)::value][j] = frag(sb + ob[k][j] + s * 16 * BRB, BRB);
    };
    auto product = [&](auto sa, auto sb) {
        constexpr int x = decltype(sa)::value, y = decltype(sb)::value;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[y][j], fa[x][i], acc[i][j], 0, 0, 0);
    };
    std::integral_constant<int, 0> S0;
    std::integral_constant<int, 1> S1;
    std::integral_constant<int, 2> S2;
    std::integral_constant<int, 3> S3;
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
        fetch_a(S0);
        fetch_b(S0);
        put_a(S0);
        put_b(S0);
    }
    fetch_a(S0);
    fetch_b(S0);
    if constexpr (SETS == 2) {
        fetch_a(S1);
        fetch_b(S1);
    }
    int slot = 0;
    wait_lds();
    meet();
    if constexpr (SPLIT) {
        // the loop of gemm_rows' split operands
        read_a(S2, 2, smem, 0);
        read_b(S0, 0, smem, 0);
        read_b(S2, 2, smem, 0);
        read_a(S1, 1, smem, 0);
        read_b(S1, 1, smem, 0);
        for (int t = 0; t < nk; ++t) {
            read_a(S0, 0, smem + slot * STAGE, 0);
            product(S2, S0);
            spread<MI * NJ, 2 * MI, 0>();
            __builtin_amdgcn_sched_barrier(0);
            slot = slot + 1 == SLOTS ? 0 : slot + 1;
            wait_lds();                                       // this stage is read, and the next one written
            meet();
            const char* nb = smem + slot * STAGE;
            read_a(S2, 2, nb, 0);
            product(S0, S2);
            spread<MI * NJ, 2 * MI, 0>();
            __builtin_amdgcn_sched_barrier(0);
            read_b(S3, 0, nb, 0);
            product(S1, S1);
            spread<MI * NJ, 2 * NJ, 0>();
            __builtin_amdgcn_sched_barrier(0);
            read_b(S2, 2, nb, 0);
            put_a(S0);
            fetch_a(S0);
            product(S1, S0);
            refill<MI * NJ, 2 * NJ, NA>();
            __builtin_amdgcn_sched_barrier(0);
            read_a(S1, 1, nb, 0);
            put_b(S0);
            fetch_b(S0);
            product(S0, S1);
            refill<MI * NJ, 2 * MI, NB>();
            __builtin_amdgcn_sched_barrier(0);
            read_b(S1, 1, nb, 0);
            product(S0, S0);
            spread<MI * NJ, 2 * NJ, 0>();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < NJ; ++j) fb[0][j] = fb[3][j];
        }
    } else {
        read_a(S0, 0, smem, 0);
        read_b(S0, 0, smem, 0);
        constexpr int READS = 2 * (MI + NJ);
        auto stage = [&](auto set) {
            const char* cb = smem + slot * STAGE;
            read_a(S1, 0, cb, 1);
            read_b(S1, 0, cb, 1);
            put_a(set);
            put_b(set);
            product(S0, S0);
            refill<MI * NJ, READS, 0, NGL>();
            __builtin_amdgcn_sched_barrier(0);
            slot = slot + 1 == SLOTS ? 0 : slot + 1;
            wait_lds();                                       // this stage is read, and the next one written
            meet();
            const char* nb = smem + slot * STAGE;
            read_a(S0, 0, nb, 0);
            read_b(S0, 0, nb, 0);
            fetch_a(set);
            fetch_b(set);
            product(S1, S1);
            refill<MI * NJ, READS, NGL, 0>();
            __builtin_amdgcn_sched_barrier(0);
        };
        for (int t = 0; t < nk; t += 2) {                     // (an odd one out is followed by a stage of zeros)
            stage(S0);
            stage(S1);
        }
    }
    // a lane's results of a 32 x 32 block: row lane & 31, element r = column (r & 3) + 8 (r >> 2) + 4 (lane >> 5)
    float* out = p.slab + (long long)zz * p.M * p.N;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int r0 = opaque(m0 + wr * RW + i * 32) + wh.r4, c0 = opaque(n0 + wc * CW + j * 32) + 4 * wh.p4;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = acc[i][j][8 * q + e];
                u32x4 a, b;
                wh.turn(raw4(v), wh.lh, raw4(v + 4), 2 + wh.lh, a, b);
                const int n = c0 + 16 * q;
                if (n >= p.N) continue;
                if (r0 < p.M) put_f32(out + (long long)r0 * p.N + n, a, n, p.N);
                if (r0 + 16 < p.M) put_f32(out + (long long)(r0 + 16) * p.N + n, b, n, p.N);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
}

}  // namespace btvae_block
