// Gated residual block: packing of operands, launches of the products in block_gemm.h, the forms for few rows, 8-bit
// quantisation and the column sums.
//
//   a = x Wg^T + bg,  b = x Wu^T + bu,  h = act(a) b,  y = h Wd^T + bd
//   dh = dy Wd,  da = dh b act'(a),  db = dh act(a),  dx = [da db] [Wg; Wu],  d[Wg; Wu] = [da db]^T x,  dWd = dy^T h
#include "block_launch.h"

using namespace btvae;
namespace bk = btvae_block;

namespace btvae_block {

// 8 consecutive values from element offset o, of which `left` exist (zeros behind them); any alignment of whole elements
template <bool SRC16> __device__ __forceinline__ void load8(const void* src, long long o, int left, float (&v)[8]) {
    if (left >= 8) {
        if (SRC16) {
            const u32x4 u = *reinterpret_cast<const u32x4_any*>(reinterpret_cast<const unsigned short*>(src) + o);
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[2 * e] = bf_lo(u[e]); v[2 * e + 1] = bf_hi(u[e]); }
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4_any*>(reinterpret_cast<const float*>(src) + o), b = *reinterpret_cast<const f32x4_any*>(reinterpret_cast<const float*>(src) + o + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? (SRC16 ? bf_load(src, o + e) : reinterpret_cast<const float*>(src)[o + e]) : 0.f;
}

// ---- operands ---------------------------------------------------------------------------------------------------------
// 8 columns c .. c + 7 of a row, as bf16 or split
template <bool SPLIT> __device__ __forceinline__ void put_operand(char* row, int c, const float (&v)[8]) {
    if constexpr (SPLIT) {
        u32x4 p[3];
        split8(v, p);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x4*>(row + split_at(c, k)) = p[k];
    } else {
        *reinterpret_cast<u32x4*>(row + 2LL * c) = pack8(v);
    }
}
// Up to four matrices become operands in one launch (a small unit's time is its launches): each takes a run of workgroups.
struct PackJob {
    const void* src; char* dst; long long ld, dld;
    int src16, planes, rows, cols, dst_cols, transpose;
    unsigned first, blocks;
};
struct PackJobs { PackJob j[4]; int n; };

// dst[r][c] = src[r][c], zeros for cols <= c < dst_cols; eight columns to a thread, `dld` bytes to a row
template <bool SRC16, bool SPLIT>
__device__ __forceinline__ void pack_rows(const PackJob& p, unsigned block) {
    const int groups = p.dst_cols / 8;
    const long long total = (long long)p.rows * groups;
    for (long long g = (long long)block * 256 + threadIdx.x; g < total; g += (long long)p.blocks * 256) {
        const long long r = g / groups;
        const int c = (int)(g - r * groups) * 8;
        float v[8];
        load8<SRC16>(p.src, r * p.ld + c, p.cols - c, v);
        put_operand<SPLIT>(p.dst + r * p.dld, c, v);
    }
}
// dst[c][r] = src[r][c] for c < cols, zeros for rows <= r < dst_cols: a 64 x 64 tile through LDS
template <bool SRC16, bool SPLIT>
__device__ __forceinline__ void pack_transposed(const PackJob& p, unsigned block, float (*t)[65]) {
    const unsigned across = (unsigned)(p.dst_cols + 63) / 64;
    const int r0 = (int)(block % across) * 64, c0 = (int)(block / across) * 64;
    float x[16];                                              // (all loads on their way together, from the first element where there is none)
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int r = r0 + 4 * k + (int)(threadIdx.x >> 6), c = c0 + (int)(threadIdx.x & 63);
        const bool in = r < p.rows && c < p.cols;
        const long long o = in ? (long long)r * p.ld + c : 0;
        x[k] = 0.f;
        if (p.rows > 0) x[k] = SRC16 ? bf_load(p.src, o) : reinterpret_cast<const float*>(p.src)[o];
        if (!in) x[k] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) t[4 * k + (threadIdx.x >> 6)][threadIdx.x & 63] = x[k];
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 8; i += 256) {
        const int c = i >> 3, rg = (i & 7) * 8;
        if (c0 + c >= p.cols || r0 + rg >= p.dst_cols) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = t[rg + e][c];
        put_operand<SPLIT>(p.dst + (long long)(c0 + c) * p.dld, r0 + rg, v);
    }
}
__global__ __launch_bounds__(256) void pack(const PackJobs jobs) {
    __shared__ float t[64][65];
    int i = 0;
    while (i + 1 < jobs.n && blockIdx.x >= jobs.j[i + 1].first) ++i;
    const PackJob p = jobs.j[i];
    const unsigned block = blockIdx.x - p.first;
    switch ((p.transpose ? 4 : 0) | (p.src16 ? 2 : 0) | (p.planes == 3 ? 1 : 0)) {
        case 0: pack_rows<false, false>(p, block); break;
        case 1: pack_rows<false, true>(p, block); break;
        case 2: pack_rows<true, false>(p, block); break;
        case 3: pack_rows<true, true>(p, block); break;
        case 4: pack_transposed<false, false>(p, block, t); break;
        case 5: pack_transposed<false, true>(p, block, t); break;
        case 6: pack_transposed<true, false>(p, block, t); break;
        default: pack_transposed<true, true>(p, block, t); break;
    }
}

// ---- partial results ------------------------------------------------------------------------------------------------
// out(m, n) (+)= sum_z slab[z][m][n] (+ bias[n]), in the order of z.  Rows [0, rows0) go to out0, [off1, off1 + rows1) to out1.
struct SlabJob {
    const float* slab; int nz, M, N;
    void* out0; long long ld; int rows0; void* out1; int off1, rows1;
    const void* bias; int bias_bf16, out_bf16, accumulate;
    unsigned first, blocks;
};
struct SlabJobs { SlabJob j[2]; int n; };
__global__ __launch_bounds__(256) void reduce_slabs(const SlabJobs jobs) {
    const SlabJob& p = jobs.j[jobs.n > 1 && blockIdx.x >= jobs.j[1].first];
    const long long total = (long long)p.M * p.N;
    for (long long i = (long long)(blockIdx.x - p.first) * 256 + threadIdx.x; i < total; i += (long long)p.blocks * 256) {
        const int m = (int)(i / p.N), n = (int)(i - (long long)m * p.N);
        void* out = p.out0;
        int row = m;
        if (m >= p.rows0) {
            row = m - p.off1;
            if (!p.out1 || row < 0 || row >= p.rows1) continue;
            out = p.out1;
        }
        float v = 0.f;
        for (int z = 0; z < p.nz; ++z) v += p.slab[(long long)z * total + i];
        if (p.bias) v += p.bias_bf16 ? bf_load(p.bias, n) : reinterpret_cast<const float*>(p.bias)[n];
        const long long o = (long long)row * p.ld + n;
        if (p.out_bf16) {
            unsigned short* d = reinterpret_cast<unsigned short*>(out);
            d[o] = bf_bits(p.accumulate ? bf_load(d, o) + v : v);
        } else {
            float* d = reinterpret_cast<float*>(out);
            d[o] = p.accumulate ? d[o] + v : v;
        }
    }
}

// part[chunk][n] = sum of src[r][n] over the chunk's rows: 64 columns x 4 row lanes to a workgroup
template <bool SRC16>
__global__ __launch_bounds__(256) void colsum_chunks(const void* __restrict__ src, long long ld, float* __restrict__ part, int rows, int N, int chunk) {
    __shared__ float red[4][64];
    const int c = (int)blockIdx.x * 64 + (threadIdx.x & 63), rl = threadIdx.x >> 6;
    const int r0 = (int)blockIdx.y * chunk, r1 = min(rows, r0 + chunk);
    float s = 0.f;
    if (c < N) {
#pragma unroll 8
        for (int r = r0 + rl; r < r1; r += 4) s += SRC16 ? bf_load(src, (long long)r * ld + c) : reinterpret_cast<const float*>(src)[(long long)r * ld + c];
    }
    red[rl][threadIdx.x & 63] = s;
    __syncthreads();
    if (rl == 0 && c < N) part[(long long)blockIdx.y * N + c] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// out0 / out1 [n] (+)= sum over strips of part[strip][0 / 1][n] (halves = 1: part[strip][n], out0 only): 32 columns x 8 strip lanes
__global__ __launch_bounds__(256) void strip_sums(const float* __restrict__ part, int strips, int N, int halves, void* out0, void* out1, int out_bf16, int accumulate) {
    __shared__ float red[8][33];
    const int cols = N * halves;
    const int c = (int)blockIdx.x * 32 + (threadIdx.x & 31), sl = threadIdx.x >> 5;
    float s = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int r = sl; r < strips; r += 8) s += part[(long long)r * cols + c];
    }
    red[sl][threadIdx.x & 31] = s;
    __syncthreads();
    if (sl != 0 || c >= cols) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x & 31];
    void* out = c < N ? out0 : out1;
    const int o = c < N ? c : c - N;
    if (!out) return;
    if (out_bf16) {
        unsigned short* d = reinterpret_cast<unsigned short*>(out);
        d[o] = bf_bits(accumulate ? bf_load(d, o) + s : s);
    } else {
        float* d = reinterpret_cast<float*>(out);
        d[o] = accumulate ? d[o] + s : s;
    }
}

// ---- 8-bit quantisation -----------------------------------------------------------------------------------------------
// Rows: one power-of-two scale for each row and 128 columns; 16 lanes x 8 values to a block.  Scaling by a power of two is
// exact, so the only rounding is the one to e4m3.  A non-finite value becomes NaN and takes no part in its block's maximum.
template <bool SRC16>
__global__ __launch_bounds__(256) void quantize_rows(const void* __restrict__ src, long long ld, unsigned char* __restrict__ q, long long ldq,
                                                     unsigned char* __restrict__ sc, long long scp, int rows, int K, int kb_n) {
    const long long total = (long long)rows * kb_n;
    for (long long g = ((long long)blockIdx.x * 256 + threadIdx.x) >> 4; g < total; g += (long long)gridDim.x * 16) {
        const long long r = g / kb_n;
        const int kb = (int)(g - r * kb_n), k = kb * 128 + (threadIdx.x & 15) * 8;
        float v[8];
        load8<SRC16>(src, r * ld + k, K - k, v);
        float mx = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, finite_abs(v[e]));
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 16));
        const int ex = scale_exp(mx);
        const float s = pow2i(-ex);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = nan_if_not_finite(v[e]) * s;
        *reinterpret_cast<u32x2*>(q + r * ldq + k) = u32x2{pack_e4m3(v[0], v[1], v[2], v[3]), pack_e4m3(v[4], v[5], v[6], v[7])};
        if ((threadIdx.x & 15) == 0) sc[r * scp + kb] = (unsigned char)(ex + 127);
    }
}

// Weights: one scale for each 128 x 128 block, one workgroup to a block
template <bool SRC16>
__global__ __launch_bounds__(256) void quantize_blocks(const void* __restrict__ src, long long ld, unsigned char* __restrict__ q, long long ldq,
                                                       unsigned char* __restrict__ sc, long long scp, int N, int K) {
    __shared__ float red[4];
    const int n0 = (int)blockIdx.y * 128, k = (int)blockIdx.x * 128 + (threadIdx.x & 15) * 8;
    auto load = [&](int n, float (&v)[8]) { load8<SRC16>(src, (long long)n * ld + k, n < N ? K - k : 0, v); };
    float mx = 0.f, v[8];
    for (int i = threadIdx.x >> 4; i < 128; i += 16) {
        load(n0 + i, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, finite_abs(v[e]));
    }
    mx = wave_max(mx);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
    __syncthreads();
    const int ex = scale_exp(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float s = pow2i(-ex);
    for (int i = threadIdx.x >> 4; i < 128 && n0 + i < N; i += 16) {
        load(n0 + i, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = nan_if_not_finite(v[e]) * s;
        *reinterpret_cast<u32x2*>(q + (long long)(n0 + i) * ldq + k) = u32x2{pack_e4m3(v[0], v[1], v[2], v[3]), pack_e4m3(v[4], v[5], v[6], v[7])};
    }
    if (threadIdx.x == 0) sc[(long long)blockIdx.y * scp + blockIdx.x] = (unsigned char)(ex + 127);
}

// values of quantised rows or blocks, as fp32
__global__ __launch_bounds__(256) void dequantize(const unsigned char* __restrict__ q, long long ldq, const unsigned char* __restrict__ sc, long long scp, int row_shift,
                                                  float* __restrict__ out, int rows, int K) {
    const long long total = (long long)rows * K;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / K;
        const int k = (int)(i - r * K);
        const float v = __builtin_amdgcn_cvt_f32_fp8((int)q[r * ldq + k], 0);
        out[i] = v * pow2i((int)sc[(r >> row_shift) * scp + (k >> 7)] - 127);
    }
}

// the same as bf16, which holds every e4m3 value times a power of two (down to 2^-126): 8 columns to a thread, whole blocks
__global__ __launch_bounds__(256) void expand_rows(const unsigned char* __restrict__ q, long long ldq, const unsigned char* __restrict__ sc, long long scp, int row_shift,
                                                   unsigned short* __restrict__ out, long long ldo, int rows, int groups) {
    const long long total = (long long)rows * groups;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / groups;
        const int k = (int)(i - r * groups) * 8;
        const u32x2 b = *reinterpret_cast<const u32x2*>(q + r * ldq + k);
        const float s = pow2i((int)sc[(r >> row_shift) * scp + (k >> 7)] - 127);
        u32x4 o;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)b[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)b[h], true);
            o[2 * h] = pack2(lo[0] * s, lo[1] * s);
            o[2 * h + 1] = pack2(hi[0] * s, hi[1] * s);
        }
        *reinterpret_cast<u32x4*>(out + r * ldo + k) = o;
    }
}

// ---- few rows -----------------------------------------------------------------------------------------------------------
// Up to 32 rows: the weights are read once, straight into the matrix instruction's registers, and the time is theirs.  A
// workgroup takes 16 weight rows (GATED: 8 gate and the 8 up rows of the same columns), its eight waves share the
// reduction in interleaved pieces and add up through LDS.  The weight rows are the MFMA's first operand, x its second.
//   fp32: v_mfma_f32_16x16x4_f32, exact products; bf16: v_mfma_f32_16x16x32_bf16, with fp32 rows x (the hidden layer of a unit, which is
//   not rounded on its way) as two bf16 pieces, off by 2^-17 of a value at most; e4m3: x quantised on the way in (every
//   workgroup repeats it: 32 values to a lane, the block's maximum over four lanes), both operands expanded to bf16, which
//   holds every e4m3 value, and multiplied as bf16: the weights' bytes are the time, and the sums are float32's.
enum { W_F32 = 0, W_BF16 = 1, W_E4M3 = 2, W_BF16_X32 = 3 };
struct FewArgs {
    const void* X; long long ldx; int x_bf16;
    const char* B; const char* B2; long long ldb;             // byte pitch
    const unsigned char* b_sc; const unsigned char* b2_sc; long long b_scp;
    const void* bias; const void* bias2; int bias_bf16;
    void* C; long long ldc; int c_bf16;
    int M, N, K, act;
};

// 32 e4m3 bytes -> 4 x 8 bf16 of the same values
__device__ __forceinline__ void expand32(const i32x8 q, bf16x8 (&o)[4]) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        u32x4 u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(q[2 * g + h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(q[2 * g + h], true);
            u[2 * h] = pack2(lo[0], lo[1]);
            u[2 * h + 1] = pack2(hi[0], hi[1]);
        }
        o[g] = __builtin_bit_cast(bf16x8, u);
    }
}

template <int WT, bool GATED, int MT, bool VEC>
__global__ __launch_bounds__(512) void gemm_few(const FewArgs p) {
    constexpr int NWV = 8, COLS = GATED ? 8 : 16;
    __shared__ float red[NWV][16][16 * MT + 1];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int row = lane & 15, kq = lane >> 4;
    const int n0 = (int)blockIdx.x * COLS;
    const int n = min(n0 + (GATED ? (row & 7) : row), p.N - 1);
    const bool up = GATED && row >= 8;
    const char* w = (up ? p.B2 : p.B) + (long long)n * p.ldb;
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const void* xr[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const long long o = (long long)min(t * 16 + row, p.M - 1) * p.ldx;
        xr[t] = p.x_bf16 ? (const void*)(reinterpret_cast<const unsigned short*>(p.X) + o) : (const void*)(reinterpret_cast<const float*>(p.X) + o);
    }

    if constexpr (WT == W_BF16) {
        constexpr int U = 4;
        auto load = [&](const void* base, int k) -> u32x4 {
            u32x4 v;
            if constexpr (VEC) {
                v = *reinterpret_cast<const u32x4*>(reinterpret_cast<const unsigned short*>(base) + min(k, p.K - 8));
                if (k >= p.K) v = u32x4{0, 0, 0, 0};
            } else {
                const unsigned short* s = reinterpret_cast<const unsigned short*>(base);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k0 = k + 2 * e, k1 = k0 + 1;
                    const unsigned lo = s[min(k0, p.K - 1)], hi = s[min(k1, p.K - 1)];
                    v[e] = (k0 < p.K ? lo : 0u) | (k1 < p.K ? hi << 16 : 0u);
                }
            }
            return v;
        };
        for (int kb = wid * 32; kb < p.K; kb += NWV * 32 * U) {
            u32x4 a[U], b[U][MT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = kb + u * NWV * 32 + kq * 8;
                a[u] = load(w, k);
#pragma unroll
                for (int t = 0; t < MT; ++t) b[u][t] = load(xr[t], k);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[u]), __builtin_bit_cast(bf16x8, b[u][t]), acc[t], 0, 0, 0);
        }
    } else if constexpr (WT == W_BF16_X32) {
        constexpr int U = 2;
        for (int kb = wid * 32; kb < p.K; kb += NWV * 32 * U) {
            u32x4 a[U];
            float b[U][MT][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = kb + u * NWV * 32 + kq * 8;
                float wv[8];
                if constexpr (VEC) {
                    a[u] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const unsigned short*>(w) + min(k, p.K - 8));
                    if (k >= p.K) a[u] = u32x4{0, 0, 0, 0};
                } else {
                    load8<true>(w, k, p.K - k, wv);
                    a[u] = pack8(wv);
                }
#pragma unroll
                for (int t = 0; t < MT; ++t) load8<false>(xr[t], k, p.K - k, b[u][t]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    float lo[8];
                    const u32x4 hi = pack8(b[u][t]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // a value that is infinite as bf16 has no second piece
                        const float h0 = bf_lo(hi[e]), h1 = bf_hi(hi[e]);
                        lo[2 * e] = __builtin_fabsf(h0) < __builtin_inff() ? b[u][t][2 * e] - h0 : 0.f;
                        lo[2 * e + 1] = __builtin_fabsf(h1) < __builtin_inff() ? b[u][t][2 * e + 1] - h1 : 0.f;
                    }
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[u]), __builtin_bit_cast(bf16x8, hi), acc[t], 0, 0, 0);
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[u]), __builtin_bit_cast(bf16x8, pack8(lo)), acc[t], 0, 0, 0);
                }
        }
    } else if constexpr (WT == W_F32) {
        constexpr int U = 8;
        auto load = [&](const void* base, int k) -> f32x4 {
            const float* s = reinterpret_cast<const float*>(base);
            f32x4 v;
            if constexpr (VEC) {
                v = *reinterpret_cast<const f32x4*>(s + min(k, p.K - 4));
                if (k >= p.K) v = f32x4{0.f, 0.f, 0.f, 0.f};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = s[min(k + e, p.K - 1)];
                    v[e] = k + e < p.K ? x : 0.f;
                }
            }
            return v;
        };
        for (int kb = wid * 16; kb < p.K; kb += NWV * 16 * U) {
            f32x4 a[U], b[U][MT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = kb + u * NWV * 16 + kq * 4;
                a[u] = load(w, k);
#pragma unroll
                for (int t = 0; t < MT; ++t) b[u][t] = load(xr[t], k);
            }
            // step e of a piece multiplies reduction elements e, 4 + e, 8 + e, 12 + e: any order will do as long as both operands agree
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u][e], b[u][t][e], acc[t], 0, 0, 0);
        }
    } else {
        const unsigned char* wsc = (GATED && kq >= 2 ? p.b2_sc : p.b_sc) + (long long)(min(n0, p.N - 1) >> 7) * p.b_scp;      // of this lane's results
        const int kbn = (p.K + 127) >> 7;
        for (int kb = wid; kb < kbn; kb += NWV) {
            const i32x4 a0 = *reinterpret_cast<const i32x4*>(w + kb * 128 + kq * 32), a1 = *reinterpret_cast<const i32x4*>(w + kb * 128 + kq * 32 + 16);
            const i32x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
            const int ew = (int)wsc[kb] - 127;
            bf16x8 wa[4];
            expand32(a, wa);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                float v[32];
                const int k = kb * 128 + kq * 32;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    if constexpr (VEC) {
                        const int kk = min(k + g * 8, p.K - 8);
                        const bool in = k + g * 8 < p.K;
                        if (p.x_bf16) {
                            const u32x4 u = *reinterpret_cast<const u32x4*>(reinterpret_cast<const unsigned short*>(xr[t]) + kk);
#pragma unroll
                            for (int e = 0; e < 4; ++e) { v[g * 8 + 2 * e] = in ? bf_lo(u[e]) : 0.f; v[g * 8 + 2 * e + 1] = in ? bf_hi(u[e]) : 0.f; }
                        } else {
                            const f32x4 u0 = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(xr[t]) + kk);
                            const f32x4 u1 = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(xr[t]) + kk + 4);
#pragma unroll
                            for (int e = 0; e < 4; ++e) { v[g * 8 + e] = in ? u0[e] : 0.f; v[g * 8 + 4 + e] = in ? u1[e] : 0.f; }
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int kk = min(k + g * 8 + e, p.K - 1);
                            const float x = p.x_bf16 ? bf_load(xr[t], kk) : reinterpret_cast<const float*>(xr[t])[kk];
                            v[g * 8 + e] = k + g * 8 + e < p.K ? x : 0.f;
                        }
                    }
                }
                float mx = 0.f;
#pragma unroll
                for (int e = 0; e < 32; ++e) mx = fmaxf(mx, finite_abs(v[e]));
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const int ex = scale_exp(mx);
                const float s = pow2i(-ex);
                i32x8 b;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    b[e] = (int)pack_e4m3(nan_if_not_finite(v[4 * e]) * s, nan_if_not_finite(v[4 * e + 1]) * s, nan_if_not_finite(v[4 * e + 2]) * s, nan_if_not_finite(v[4 * e + 3]) * s);
                bf16x8 xb[4];
                expand32(b, xb);
                f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < 4; ++g) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wa[g], xb[g], d, 0, 0, 0);
                // a lane's four results: x row lane & 15, the row it quantised; weight rows of one block (GATED: lanes 0-31 gate, 32-63 up)
                // (both scales at once: one after the other a sum may leave float32's range on its way)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] += __builtin_amdgcn_ldexpf(d[i], ex + ew);
            }
        }
    }
    // element i of a lane: weight row 4 (lane >> 4) + i, x row lane & 15
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wid][4 * kq + i][t * 16 + row] = acc[t][i];
    __syncthreads();
    for (int i = tid; i < COLS * 16 * MT; i += 512) {
        const int c = i % COLS, m = i / COLS, nn = n0 + c;
        if (m >= p.M || nn >= p.N) continue;
        float v = 0.f, u = 0.f;
#pragma unroll
        for (int q = 0; q < NWV; ++q) {
            v += red[q][c][m];
            if (GATED) u += red[q][c + 8][m];
        }
        if (p.bias) v += p.bias_bf16 ? bf_load(p.bias, nn) : reinterpret_cast<const float*>(p.bias)[nn];
        if (GATED) {
            if (p.bias2) u += p.bias_bf16 ? bf_load(p.bias2, nn) : reinterpret_cast<const float*>(p.bias2)[nn];
            float a, d;
            with_act(p.act, [&](auto act) { act_value<false, decltype(act)::value>(p.act, v, a, d); });
            v = a * u;
        }
        const long long o = (long long)m * p.ldc + nn;
        if (p.c_bf16) reinterpret_cast<unsigned short*>(p.C)[o] = bf_bits(v);
        else reinterpret_cast<float*>(p.C)[o] = v;
    }
}

// ---- launches ---------------------------------------------------------------------------------------------------------
// Splits of a reduction of `stages` stages over fewer tiles than compute units: as many as fill the chip about once, each at least
// 12 stages long (the ring's fill and the slab's write and read cost about that much).
inline int row_splits(int T, int stages, int unit) {
    if (T <= 0 || T >= CHIP * 3 / 4) return 1;
    int z = std::min(CHIP / T, stages / std::max(12, unit));
    return std::max(1, std::min(z, 32));
}

struct ProductPlan { int z, kz; };
// EP_LINEAR: splits of the reduction, each a multiple of `unit` stages; tiles of 128 x `tn`
static ProductPlan plan_product(int M, int N, int tn, int stages, int unit) {
    if (M <= 0 || N <= 0 || stages <= 0) return {1, std::max(1, stages)};
    ProductPlan r;
    r.kz = tiles(tiles(stages, row_splits(tiles(M, 128) * tiles(N, tn), stages, unit)), unit) * unit;
    r.z = tiles(stages, r.kz);
    return r;
}
// Launch of reduce_slabs over one or two results
static int launch_reduce(SlabJobs& q, hipStream_t s, const char* what) {
    unsigned blocks = 0;
    for (int i = 0; i < q.n; ++i) {
        q.j[i].first = blocks;
        q.j[i].blocks = (unsigned)std::min<long long>(((long long)q.j[i].M * q.j[i].N + 255) / 256, 8192);
        blocks += q.j[i].blocks;
    }
    hipLaunchKernelGGL(reduce_slabs, dim3(blocks), dim3(256), 0, s, q);
    return btvae::check_launch(what);
}
struct ColPlan { int big, z, rz; };
// `beside`: tiles of another product in the same launch
static ColPlan plan_cols(int M, int N, int R, int beside = 0) {
    ColPlan r;
    // 256 x 256 tiles from where their splits fill the chip: see gemm_cols
    r.big = !beside && tiles(M, 256) * tiles(N, 256) * std::max(1, R / 1024) >= CHIP;
    const int t = r.big ? 256 : 128;
    const int T = std::max(1, tiles(M, t) * tiles(N, t) + beside);
    // fill the chip; a split has at least 256 rows, and multiples of eight splits keep one row range on one XCD
    const int fill = r.big ? CHIP : 2 * CHIP;
    int z = std::max(1, std::min((T >= fill ? 1 : fill / T), tiles(R, 256)));
    if (z > 8) z = z / 8 * 8;
    const int cap = 1 << 20;                                          // rows of a split
    z = std::max(z, tiles(R, cap));
    r.rz = tiles(tiles(std::max(R, 1), z), 32) * 32;
    r.z = std::max(1, tiles(R, r.rz));
    return r;
}

}  // namespace btvae_block

#define BLK_STREAM(s) reinterpret_cast<hipStream_t>(s)

// Operand matrices: bf16 (planes 1), or split (planes 3: 96 bytes for every 16 columns).  `ld` bytes to a row, rows on 16 bytes.
static bool operand_ok(const void* p, long long ld, int planes, int cols) {
    return bk::al16(p) && (ld & 15) == 0 && ld >= (planes == 3 ? (long long)bk::tiles(cols, 16) * 96 : 2LL * cols);
}
static int stages_of(int K, int planes) { return planes == 3 ? bk::tiles(K, 16) : bk::tiles(K, 64); }

// n <= 4 jobs of ten numbers: src, src_bf16, ld, dst, planes, dst_ld, rows, cols, dst_cols, transpose
BTVAE_API int btvae_block_pack(const long long* jobs, int n, void* stream) {
    BTVAE_REQUIRE(jobs && n >= 0 && n <= 4, "block_pack: up to four matrices");
    bk::PackJobs q;
    q.n = 0;
    long long blocks = 0;
    for (int i = 0; i < n; ++i) {
        const long long* a = jobs + 10 * i;
        bk::PackJob p;
        p.src = reinterpret_cast<const void*>(a[0]); p.src16 = a[1] != 0; p.ld = a[2];
        p.dst = reinterpret_cast<char*>(a[3]); p.planes = (int)a[4]; p.dld = a[5];
        BTVAE_REQUIRE(a[6] >= 0 && a[7] > 0 && a[8] > 0 && a[6] < (1LL << 31) && a[7] < (1LL << 31) && a[8] < (1LL << 31) && p.ld >= a[7], "block_pack: bad source shape");
        p.rows = (int)a[6]; p.cols = (int)a[7]; p.dst_cols = (int)a[8]; p.transpose = a[9] != 0;
        BTVAE_REQUIRE(p.planes == 1 || p.planes == 3, "block_pack: planes must be 1 or 3");
        BTVAE_REQUIRE((p.dst_cols & 15) == 0 && p.dst_cols >= (p.transpose ? p.rows : p.cols) && operand_ok(p.dst, p.dld, p.planes, p.dst_cols), "block_pack: bad destination layout");
        if (p.rows == 0 && !p.transpose) continue;
        BTVAE_REQUIRE((p.src || p.rows == 0) && p.dst, "block_pack: null matrix");
        const long long b = p.transpose ? (long long)bk::tiles(p.dst_cols, 64) * bk::tiles(p.cols, 64) : std::min<long long>(((long long)p.rows * (p.dst_cols / 8) + 255) / 256, 16384);
        p.first = (unsigned)blocks; p.blocks = (unsigned)b;
        blocks += b;
        BTVAE_REQUIRE(blocks < (1LL << 31), "block_pack: too large");
        q.j[q.n++] = p;
    }
    if (q.n == 0) return 0;
    hipLaunchKernelGGL(bk::pack, dim3((unsigned)blocks), dim3(256), 0, BLK_STREAM(stream), q);
    return check_launch("block_pack");
}

// Bytes of the kept projections: blocks of 32 x 32 values of a and of b, 24 bits a value for bf16 operands, else 32
BTVAE_API long long btvae_gated_kept_bytes(int M, int F, int planes) {
    return (long long)bk::tiles(M, 32) * bk::tiles(F, 32) * 2 * (planes == 3 ? bk::kept_bytes<false>() : bk::kept_bytes<true>());
}
BTVAE_API int btvae_gated_proj_fwd(const void* X, long long ldx, const void* Wg, const void* Wu, long long ldw, const void* bg, const void* bu, int bias_bf16,
                                   void* H, long long ldh, void* kept, int planes, int act, int M, int F, int K, void* stream) {
    BTVAE_REQUIRE(planes == 1 || planes == 3, "gated_proj_fwd: planes must be 1 or 3");
    BTVAE_REQUIRE(M >= 0 && F > 0 && K > 0 && (planes == 3 || (K & 7) == 0), "gated_proj_fwd: bad sizes (M %d, F %d, K %d)", M, F, K);
    BTVAE_REQUIRE(act >= 0 && act <= 3, "gated_proj_fwd: unknown activation %d", act);
    if (M == 0) return 0;
    BTVAE_REQUIRE(operand_ok(X, ldx, planes, K) && operand_ok(Wg, ldw, planes, K) && operand_ok(Wu, ldw, planes, K), "gated_proj_fwd: bad operand layout");
    BTVAE_REQUIRE(operand_ok(H, ldh, planes, bk::tiles(F, 16) * 16) && ldh < (1 << 24), "gated_proj_fwd: bad layout of H");
    BTVAE_REQUIRE(bk::al16(kept), "gated_proj_fwd: the kept projections must start on 16 bytes");
    bk::Args p = {};
    p.A = (const char*)X; p.lda = ldx; p.B = (const char*)Wg; p.B2 = (const char*)Wu; p.ldb = ldw;
    p.M = M; p.N = F; p.K = K; p.ks = p.kz = stages_of(K, planes);
    p.bias = bg; p.bias2 = bu; p.bias_bf16 = bias_bf16;
    p.C = H; p.ldc = planes == 3 ? ldh : ldh / 2;
    p.act = act; p.kept = (char*)kept; p.half = bk::tiles(F, 32) * 32;
    ProfScope prof(PK_GEMM_FWD, BLK_STREAM(stream), 4.0 * M * F * K, 0.0);
    if (planes == 3) return bk::launch_rows<bk::FMT_SPLIT, bk::EP_GATED_3>(p, 1, BLK_STREAM(stream), "gated_proj_fwd");
    return bk::launch_rows<bk::FMT_BF16, bk::EP_GATED>(p, 1, BLK_STREAM(stream), "gated_proj_fwd");
}

BTVAE_API int btvae_gated_proj_bwd(const void* dY, long long lddy, const void* WdT, long long ldw, const void* kept, void* dGU, long long ldd, float* colpart, int planes, int act, int M, int F, int N, void* stream) {
    BTVAE_REQUIRE(planes == 1 || planes == 3, "gated_proj_bwd: planes must be 1 or 3");
    BTVAE_REQUIRE(M >= 0 && F > 0 && N > 0 && (planes == 3 || (N & 7) == 0), "gated_proj_bwd: bad sizes (M %d, F %d, N %d)", M, F, N);
    BTVAE_REQUIRE(act >= 0 && act <= 3, "gated_proj_bwd: unknown activation %d", act);
    if (M == 0) return 0;
    BTVAE_REQUIRE(operand_ok(dY, lddy, planes, N) && operand_ok(WdT, ldw, planes, N), "gated_proj_bwd: bad operand layout");
    const int half = bk::tiles(F, 32) * 32;
    BTVAE_REQUIRE(kept && bk::al16(kept), "gated_proj_bwd: the kept projections must start on 16 bytes");
    BTVAE_REQUIRE(operand_ok(dGU, ldd, planes, 2 * half) && ldd < (1 << 26), "gated_proj_bwd: bad layout of the gradients");
    bk::Args p = {};
    p.A = (const char*)dY; p.lda = lddy; p.B = (const char*)WdT; p.ldb = ldw;
    p.M = M; p.N = F; p.K = N; p.ks = p.kz = stages_of(N, planes);
    p.C = dGU; p.ldc = planes == 3 ? ldd : ldd / 2;
    p.act = act; p.kept = (char*)const_cast<void*>(kept); p.half = half; p.colpart = colpart;
    ProfScope prof(PK_GEMM_DGRAD, BLK_STREAM(stream), 2.0 * M * F * N, 0.0);
    if (planes == 3) return bk::launch_rows<bk::FMT_SPLIT, bk::EP_GATED_BWD_3>(p, 1, BLK_STREAM(stream), "gated_proj_bwd");
    return bk::launch_rows<bk::FMT_BF16, bk::EP_GATED_BWD>(p, 1, BLK_STREAM(stream), "gated_proj_bwd");
}
// Strips of rows that btvae_gated_proj_bwd leaves column sums for: colpart holds [strips][2][F] floats.
BTVAE_API int btvae_gated_proj_strips(int M) { return 2 * bk::tiles(M, 128); }

BTVAE_API long long btvae_block_product_ws(int M, int N, int K, int planes) {
    const bk::ProductPlan r = bk::plan_product(M, N, bk::tile_width(planes == 3), stages_of(K, planes), 1);
    return r.z > 1 ? (long long)r.z * M * N : 0;
}
BTVAE_API int btvae_block_product(const void* A, long long lda, const void* B, long long ldb, const void* bias, int bias_bf16, void* C, long long ldc, int c_bf16,
                                  float* ws, long long ws_floats, int planes, int M, int N, int K, void* stream) {
    BTVAE_REQUIRE(planes == 1 || planes == 3, "block_product: planes must be 1 or 3");
    BTVAE_REQUIRE(M >= 0 && N > 0 && K > 0 && (planes == 3 || (K & 7) == 0) && ldc >= N, "block_product: bad sizes (M %d, N %d, K %d)", M, N, K);
    if (M == 0) return 0;
    BTVAE_REQUIRE(operand_ok(A, lda, planes, K) && operand_ok(B, ldb, planes, K), "block_product: bad operand layout");
    hipStream_t s = BLK_STREAM(stream);
    bk::Args p = {};
    p.A = (const char*)A; p.lda = lda; p.B = (const char*)B; p.ldb = ldb;
    p.M = M; p.N = N; p.K = K; p.ks = stages_of(K, planes);
    const bk::ProductPlan r = bk::plan_product(M, N, bk::tile_width(planes == 3), p.ks, 1);
    BTVAE_REQUIRE(r.z == 1 || (ws && ws_floats >= (long long)r.z * M * N), "block_product: workspace too small");
    p.kz = r.kz; p.slab = ws;
    p.bias = bias; p.bias_bf16 = bias_bf16;
    p.C = C; p.ldc = ldc; p.c_type = c_bf16 ? bk::T_BF16 : bk::T_F32;
    ProfScope prof(PK_GEMM_FWD, s, 2.0 * M * N * K, 0.0);
    const int rc = planes == 3 ? bk::launch_rows<bk::FMT_SPLIT, bk::EP_LINEAR>(p, r.z, s, "block_product") : bk::launch_rows<bk::FMT_BF16, bk::EP_LINEAR>(p, r.z, s, "block_product");
    if (rc || r.z == 1) return rc;
    bk::SlabJobs q = {};
    q.n = 1;
    q.j[0] = {ws, r.z, M, N, C, ldc, M, nullptr, 0, 0, bias, bias_bf16, c_bf16, 0, 0, 0};
    return bk::launch_reduce(q, s, "block_product reduction");
}

namespace btvae_block {
struct ColJob {
    const void* A; long long lda; const void* B; long long ldb;
    void* out0; long long rows0; void* out1; long long off1, rows1, ldo, out_bf16; long long M, N;
};
static int tiles128(const ColJob& j) { return tiles((int)j.M, 128) * tiles((int)j.N, 128); }
// Two products in one launch where both are small enough for 128 x 128 tiles and all their splits are on the chip at a time (measured:
// the three weight gradients of 203 x 531 from 1537 rows, fp32: 17 + 4 + 15 + 4 us in four launches, 18 + 5 in two)
static bool side_by_side(const ColJob& a, const ColJob& b, int R) {
    return !plan_cols((int)a.M, (int)a.N, R).big && !plan_cols((int)b.M, (int)b.N, R).big && tiles128(a) + tiles128(b) <= 2 * CHIP;
}
static long long cols_floats(const ColJob& j, int z) { return (long long)z * j.M * j.N; }
static long long cols_ws(const ColJob* j, int n, int R) {
    if (n == 2 && side_by_side(j[0], j[1], R)) {
        const int z = plan_cols((int)j[0].M, (int)j[0].N, R, tiles128(j[1])).z;
        return cols_floats(j[0], z) + cols_floats(j[1], z);
    }
    long long need = 0;
    for (int i = 0; i < n; ++i) need = std::max(need, cols_floats(j[i], plan_cols((int)j[i].M, (int)j[i].N, R).z));
    return need;
}
static int run_cols(const ColJob* j, int n, float* ws, int planes, int R, int accumulate, hipStream_t s) {
    const int unit = planes == 3 ? 16 : 8;
    const ColPlan r = n == 2 ? plan_cols((int)j[0].M, (int)j[0].N, R, tiles128(j[1])) : plan_cols((int)j[0].M, (int)j[0].N, R);
    const int t = r.big ? 256 : 128;
    ColPair q = {};
    SlabJobs sums = {};
    sums.n = n;
    float* slab = ws;
    double flops = 0;
    for (int i = 0; i < n; ++i) {
        ColArgs& p = q.a[i];
        const int M = (int)j[i].M, N = (int)j[i].N;
        p.A = (const char*)j[i].A; p.lda = j[i].lda; p.a_cols = tiles(M, unit) * unit; p.B = (const char*)j[i].B; p.ldb = j[i].ldb; p.b_cols = tiles(N, unit) * unit;
        p.R = R; p.M = M; p.N = N; p.rz = r.rz; p.slab = slab; p.tiles_m = tiles(M, t); p.tiles_n = tiles(N, t);
        if (i == 0) q.tiles0 = p.tiles_m * p.tiles_n;
        q.tiles += p.tiles_m * p.tiles_n;
        sums.j[i] = {slab, r.z, M, N, j[i].out0, j[i].ldo, (int)j[i].rows0, j[i].out1, (int)j[i].off1, (int)j[i].rows1, nullptr, 0, (int)j[i].out_bf16, accumulate, 0, 0};
        slab += cols_floats(j[i], r.z);
        flops += 2.0 * M * N * R;
    }
    {
        ProfScope prof(PK_GEMM_WGRAD, s, flops, 0.0);
        if (int rc = launch_cols(q, planes == 3, r.big, r.z, s)) return rc;
    }
    return launch_reduce(sums, s, "block_wgrad reduction");
}
}  // namespace btvae_block

static int check_cols(const bk::ColJob& j, int planes, int R) {
    BTVAE_REQUIRE(planes == 1 || planes == 3, "block_wgrad: planes must be 1 or 3");
    BTVAE_REQUIRE(j.M > 0 && j.N > 0 && j.M < (1 << 30) && j.N < (1 << 30) && R >= 0 && j.rows0 > 0 && j.rows0 <= j.M && j.ldo >= j.N && j.out0, "block_wgrad: bad sizes (M %lld, N %lld, R %d)", j.M, j.N, R);
    const int unit = planes == 3 ? 16 : 8, M8 = bk::tiles((int)j.M, unit) * unit, N8 = bk::tiles((int)j.N, unit) * unit;
    BTVAE_REQUIRE(!j.out1 || (j.off1 >= j.rows0 && j.rows1 >= 0 && j.off1 + j.rows1 <= j.M), "block_wgrad: bad row ranges");
    BTVAE_REQUIRE(R == 0 || (operand_ok(j.A, j.lda, planes, M8) && operand_ok(j.B, j.ldb, planes, N8)), "block_wgrad: operand rows must start on 16 bytes and hold whole groups of %d columns", unit);
    BTVAE_REQUIRE(j.lda < bk::MAX_PITCH && j.ldb < bk::MAX_PITCH, "block_wgrad: rows of more than 8 MiB");
    BTVAE_REQUIRE(R <= bk::MAX_ROWS, "block_wgrad: too many rows");
    return 0;
}
BTVAE_API long long btvae_block_wgrad_ws(int M, int N, int R, int planes) {
    bk::ColJob j = {};
    j.M = M; j.N = N;
    return bk::cols_ws(&j, 1, R);
}
// out(m, n) (+)= sum_r A[r][m] B[r][n], m < M (rows [0, rows0) -> out0, [off1, off1 + rows1) -> out1), n < N
BTVAE_API int btvae_block_wgrad(const void* A, long long lda, const void* B, long long ldb, float* ws, long long ws_floats,
                                void* out0, int rows0, void* out1, int off1, int rows1, long long ldo, int out_bf16, int accumulate, int planes, int M, int N, int R, void* stream) {
    const bk::ColJob j = {A, lda, B, ldb, out0, rows0, out1, off1, rows1, ldo, out_bf16, M, N};
    if (int rc = check_cols(j, planes, R)) return rc;
    BTVAE_REQUIRE(ws && ws_floats >= bk::cols_ws(&j, 1, R), "block_wgrad: workspace too small");
    return bk::run_cols(&j, 1, ws, planes, R, accumulate, BLK_STREAM(stream));
}
// Two such sums over the same rows, in one launch where that pays: jobs of thirteen numbers (A, lda, B, ldb, out0, rows0, out1, off1, rows1, ldo, out_bf16, M, N)
static void cols_jobs(const long long* a, bk::ColJob* j) {
    for (int i = 0; i < 2; ++i, a += 13) j[i] = {(const void*)a[0], a[1], (const void*)a[2], a[3], (void*)a[4], a[5], (void*)a[6], a[7], a[8], a[9], a[10], a[11], a[12]};
}
BTVAE_API long long btvae_block_wgrad_pair_ws(int M0, int N0, int M1, int N1, int R, int planes) {
    bk::ColJob j[2] = {};
    j[0].M = M0; j[0].N = N0; j[1].M = M1; j[1].N = N1;
    return bk::cols_ws(j, 2, R);
}
BTVAE_API int btvae_block_wgrad_pair(const long long* jobs, float* ws, long long ws_floats, int planes, int R, int accumulate, void* stream) {
    BTVAE_REQUIRE(jobs, "block_wgrad: null jobs");
    bk::ColJob j[2];
    cols_jobs(jobs, j);
    for (int i = 0; i < 2; ++i)
        if (int rc = check_cols(j[i], planes, R)) return rc;
    BTVAE_REQUIRE(ws && ws_floats >= bk::cols_ws(j, 2, R), "block_wgrad: workspace too small");
    hipStream_t s = BLK_STREAM(stream);
    if (bk::side_by_side(j[0], j[1], R)) return bk::run_cols(j, 2, ws, planes, R, accumulate, s);
    if (int rc = bk::run_cols(j, 1, ws, planes, R, accumulate, s)) return rc;
    return bk::run_cols(j + 1, 1, ws, planes, R, accumulate, s);
}

// out[n] (+)= sum_r src[r][n]; ws: btvae_block_colsum_ws floats
static int colsum_chunk(int R) { return std::max(64, bk::tiles(R, 256)); }
BTVAE_API long long btvae_block_colsum_ws(int R, int N) { return (long long)std::max(1, bk::tiles(R, colsum_chunk(R))) * N; }
BTVAE_API int btvae_block_colsum(const void* src, int src_bf16, long long ld, float* ws, long long ws_floats, void* out, int out_bf16, int accumulate, int R, int N, void* stream) {
    BTVAE_REQUIRE(R >= 0 && N > 0 && (R == 0 || ld >= N) && out, "block_colsum: bad sizes (R %d, N %d)", R, N);
    BTVAE_REQUIRE(ws && ws_floats >= btvae_block_colsum_ws(R, N), "block_colsum: workspace too small");
    hipStream_t s = BLK_STREAM(stream);
    const int chunk = colsum_chunk(R), nc = bk::tiles(R, chunk);
    if (nc > 0) {
        const dim3 grid((unsigned)bk::tiles(N, 64), (unsigned)nc);
        if (src_bf16) hipLaunchKernelGGL((bk::colsum_chunks<true>), grid, dim3(256), 0, s, src, ld, ws, R, N, chunk);
        else hipLaunchKernelGGL((bk::colsum_chunks<false>), grid, dim3(256), 0, s, src, ld, ws, R, N, chunk);
        if (int rc = check_launch("block_colsum")) return rc;
    }
    hipLaunchKernelGGL(bk::strip_sums, dim3((unsigned)bk::tiles(N, 32)), dim3(256), 0, s, (const float*)ws, nc, N, 1, out, (void*)nullptr, out_bf16, accumulate);
    return check_launch("block_colsum");
}
// out0 / out1 [n] (+)= sum over strips of part[strip][0 / 1][n]
BTVAE_API int btvae_block_strip_sums(const float* part, int strips, int N, void* out0, void* out1, int out_bf16, int accumulate, void* stream) {
    BTVAE_REQUIRE(strips >= 0 && N > 0 && out0, "block_strip_sums: bad sizes");
    hipLaunchKernelGGL(bk::strip_sums, dim3((unsigned)bk::tiles(2 * N, 32)), dim3(256), 0, BLK_STREAM(stream), part, strips, N, 2, out0, out1, out_bf16, accumulate);
    return check_launch("block_strip_sums");
}

// ---- the whole unit in one call: operands laid out, projections, products, in memory that the caller gives ----
// (a unit of a few hundred rows is its host's work: six calls and eight allocations from Python cost more than its kernels)
namespace btvae_block {
struct Unit {
    const void* x; int x16; long long ldx; int M, K, F, N;
    const void *wg, *wu, *wd; long long ldg, ldu, ldd; int w16;
    const void *bg, *bu, *bd; int b16, planes, act;
};
// Memory handed out piece by piece; without a base only counted
struct Pieces {
    char* base; long long used;
    char* take(long long n) {
        char* at = base ? base + used : nullptr;
        used += (n + 255) / 256 * 256;
        return at;
    }
};
struct Operand { const void* at; long long ld; int width; bool pack; };
// Rows or columns of a product from which a bf16 matrix whose rows do not start on 64 bytes is laid out anew: such rows cost the copies to LDS more
// requests (measured, 65,536 x 1000 times 1000 x N, in place against the copy and the product: N 512 80 and 118 us, 1024 155
// and 178, 2048 346 and 316, 4096 653 and 596; never copying costs a gated unit's training pass of 65,536 x 1000 x 2000 3 %)
constexpr long long REPACK_READS = 2048;
// Rows MAX_PITCH bytes apart and more are beyond the products' offsets, and are laid out side by side.
static bool in_place(const void* t, int t16, long long ld, int cols, int planes, long long reads) {
    if (planes != 1 || !t16 || cols % 8 || ld % 8 || !al16(t) || 2 * ld >= MAX_PITCH) return false;
    return reads < REPACK_READS || (2 * ld % 64 == 0 && ((uintptr_t)t & 63) == 0);
}
static long long bytes_of(long long cols, int planes) { return cols * (planes == 3 ? 6 : 2); }
// Pitch of an operand: whole groups of 32 columns, bf16 rows on 128 bytes (h with rows on 64 of them cost the product of 65,536 x 2000 x 1000 391 us
// instead of 330)
static long long row_pitch(int cols, int planes) { return planes == 3 ? bytes_of(tiles(cols, 32) * 32LL, 3) : bytes_of(tiles(cols, 64) * 64LL, 1); }
static Operand operand(const void* t, int t16, long long ld, int rows, int cols, int planes, bool as_is, Pieces& home) {
    if (as_is) return {t, 2 * ld, cols, false};
    const long long pitch = row_pitch(cols, planes);
    return {home.take(rows * pitch), pitch, tiles(cols, 8) * 8, true};
}
// One matrix to be laid out (transpose: its transpose, behind `offset` bytes of each row)
static void add_job(long long* jobs, int& n, const void* t, int t16, long long ld, const void* at, long long pitch, int planes, int rows, int cols, int dst_cols, int transpose) {
    long long* j = jobs + 10 * n++;
    j[0] = (long long)t; j[1] = t16; j[2] = ld; j[3] = (long long)at; j[4] = planes; j[5] = pitch; j[6] = rows; j[7] = cols; j[8] = dst_cols; j[9] = transpose;
}
// What the backward pass reads: x as an operand, h, both projections.  The same order in both passes.
struct Kept { Operand X; char* H; long long ldh; char* kept; };
static Kept lay_out(const Unit& u, bool keep, Pieces& home) {
    Kept k;
    k.X = operand(u.x, u.x16, u.ldx, u.M, u.K, u.planes, in_place(u.x, u.x16, u.ldx, u.K, u.planes, 2LL * u.F), home);
    k.ldh = row_pitch(u.F, u.planes);
    k.H = home.take(u.M * k.ldh);
    k.kept = keep ? home.take(btvae_gated_kept_bytes(u.M, u.F, u.planes)) : nullptr;
    return k;
}
struct ForwardPlan { Kept k; Operand Wg, Wu, Wd; float* ws; long long ws_floats; };
static ForwardPlan plan_forward(const Unit& u, bool keep, Pieces& store, Pieces& scratch) {
    ForwardPlan p;
    p.k = lay_out(u, keep, keep ? store : scratch);
    const bool pair = u.ldg == u.ldu && in_place(u.wg, u.w16, u.ldg, u.K, u.planes, u.M) && in_place(u.wu, u.w16, u.ldu, u.K, u.planes, u.M);
    p.Wg = operand(u.wg, u.w16, u.ldg, u.F, u.K, u.planes, pair, scratch);
    p.Wu = operand(u.wu, u.w16, u.ldu, u.F, u.K, u.planes, pair, scratch);
    p.Wd = operand(u.wd, u.w16, u.ldd, u.N, u.F, u.planes, in_place(u.wd, u.w16, u.ldd, u.F, u.planes, u.M), scratch);
    p.ws_floats = btvae_block_product_ws(u.M, u.N, p.Wd.width, u.planes);
    p.ws = (float*)scratch.take(4 * p.ws_floats);
    return p;
}
// b: dy, dy_bf16, lddy, dx, dwg, dwu, dwd, dbg, dbu, dbd, their types (w_gate and w_up, w_down, b_gate and b_up, b_down: bf16), accumulate
struct BackwardPlan {
    Operand DY, WdT, WT;
    char* dGU; long long ldd; int half;
    float *colpart, *ws, *other;
    long long dx_floats, w_floats, c_floats;
};
static BackwardPlan plan_backward(const Unit& u, const long long* b, Pieces& scratch) {
    BackwardPlan p;
    p.half = tiles(u.F, 32) * 32;
    const int n32 = tiles(u.N, 32) * 32, unit = u.planes == 3 ? 96 : 128;
    const auto up = [&](long long n) { return (n + unit - 1) / unit * unit; };
    p.DY = operand((const void*)b[0], (int)b[1], b[2], u.M, u.N, u.planes, in_place((const void*)b[0], (int)b[1], b[2], u.N, u.planes, 2LL * u.F), scratch);
    p.WdT = {nullptr, up(bytes_of(n32, u.planes)), n32, true};
    p.WdT.at = scratch.take(u.F * p.WdT.ld);
    p.WT = {nullptr, up(bytes_of(2LL * p.half, u.planes)), 2 * p.half, true};
    p.WT.at = b[3] ? scratch.take(u.K * p.WT.ld) : nullptr;
    p.ldd = bytes_of(2LL * p.half, u.planes);
    p.dGU = scratch.take(u.M * p.ldd);
    const bool weights = b[4] != 0;
    p.colpart = weights && (b[7] || b[8]) ? (float*)scratch.take(4LL * btvae_gated_proj_strips(u.M) * 2 * u.F) : nullptr;
    p.other = weights && !b[7] && b[8] ? (float*)scratch.take(4LL * u.F) : nullptr;      // (sums that nobody wants)
    // one after the other, so one place
    p.dx_floats = b[3] ? btvae_block_product_ws(u.M, u.K, 2 * p.half, u.planes) : 0;
    p.w_floats = weights ? btvae_block_wgrad_pair_ws(2 * p.half, u.K, u.N, u.F, u.M, u.planes) : 0;
    p.c_floats = weights && b[9] ? btvae_block_colsum_ws(u.M, u.N) : 0;
    p.ws = (float*)scratch.take(4 * std::max({p.dx_floats, p.w_floats, p.c_floats}));
    return p;
}
}  // namespace btvae_block

// a: x, x_bf16, ldx, M, K, F, N, wg, ldg, wu, ldu, wd, ldd, weights bf16, bg, bu, bd, biases bf16, planes, act
static int unit_of(const long long* a, bk::Unit& u) {
    BTVAE_REQUIRE(a, "gated_unit: null description");
    const long long big = 1LL << 30;
    BTVAE_REQUIRE(a[3] >= 0 && a[3] <= bk::MAX_ROWS && a[4] > 0 && a[4] < big && a[5] > 0 && a[5] < big && a[6] > 0 && a[6] < big, "gated_unit: bad sizes (M %lld, K %lld, F %lld, N %lld)", a[3], a[4], a[5], a[6]);
    BTVAE_REQUIRE(a[2] >= a[4] && a[8] >= a[4] && a[10] >= a[4] && a[12] >= a[5], "gated_unit: rows overlap");
    BTVAE_REQUIRE(a[18] == 1 || a[18] == 3, "gated_unit: planes must be 1 or 3");
    BTVAE_REQUIRE(a[19] >= 0 && a[19] <= 3, "gated_unit: unknown activation %lld", a[19]);
    BTVAE_REQUIRE((a[0] || a[3] == 0) && a[7] && a[9] && a[11], "gated_unit: null matrix");
    u = {(const void*)a[0], a[1] != 0, a[2], (int)a[3], (int)a[4], (int)a[5], (int)a[6], (const void*)a[7], (const void*)a[9], (const void*)a[11], a[8], a[10], a[12], a[13] != 0,
         (const void*)a[14], (const void*)a[15], (const void*)a[16], a[17] != 0, (int)a[18], (int)a[19]};
    return 0;
}
// bytes[0]: what the backward pass needs kept (0 without `keep`), bytes[1]: scratch of the forward pass, bytes[2]: 1 if x is read where it is
BTVAE_API int btvae_gated_unit_bytes(const long long* unit, int keep, long long* bytes) {
    bk::Unit u;
    if (int rc = unit_of(unit, u)) return rc;
    bk::Pieces store = {nullptr, 0}, scratch = {nullptr, 0};
    const bk::ForwardPlan p = bk::plan_forward(u, keep != 0, store, scratch);
    bytes[0] = store.used; bytes[1] = scratch.used; bytes[2] = !p.k.X.pack;
    return 0;
}
BTVAE_API int btvae_gated_unit_fwd(const long long* unit, void* y, long long ldy, int y_bf16, void* store, long long store_bytes, void* scratch, long long scratch_bytes, void* stream) {
    bk::Unit u;
    if (int rc = unit_of(unit, u)) return rc;
    if (u.M == 0) return 0;
    bk::Pieces kept = {(char*)store, 0}, spare = {(char*)scratch, 0};
    const bk::ForwardPlan p = bk::plan_forward(u, store != nullptr, kept, spare);
    BTVAE_REQUIRE(kept.used <= store_bytes && spare.used <= scratch_bytes && (scratch || spare.used == 0), "gated_unit: workspace too small");
    long long jobs[40];
    int n = 0;
    const auto pack = [&](const bk::Operand& o, const void* t, int t16, long long ld, int rows, int cols) {
        if (o.pack) bk::add_job(jobs, n, t, t16, ld, o.at, o.ld, u.planes, rows, cols, bk::tiles(cols, 32) * 32, 0);
    };
    pack(p.k.X, u.x, u.x16, u.ldx, u.M, u.K);
    pack(p.Wg, u.wg, u.w16, u.ldg, u.F, u.K);
    pack(p.Wu, u.wu, u.w16, u.ldu, u.F, u.K);
    pack(p.Wd, u.wd, u.w16, u.ldd, u.N, u.F);
    if (int rc = btvae_block_pack(jobs, n, stream)) return rc;
    if (int rc = btvae_gated_proj_fwd(p.k.X.at, p.k.X.ld, p.Wg.at, p.Wu.at, p.Wg.ld, u.bg, u.bu, u.b16, p.k.H, p.k.ldh, p.k.kept, u.planes, u.act, u.M, u.F, p.k.X.width, stream)) return rc;
    return btvae_block_product(p.k.H, p.k.ldh, p.Wd.at, p.Wd.ld, u.bd, u.b16, y, ldy, y_bf16, p.ws, p.ws_floats, u.planes, u.M, u.N, p.Wd.width, stream);
}
static int check_back(const bk::Unit& u, const long long* b) {
    BTVAE_REQUIRE(b && (b[0] || u.M == 0) && b[2] >= u.N, "gated_unit: bad gradient of the result");
    BTVAE_REQUIRE((b[4] != 0) == (b[5] != 0) && (b[4] != 0) == (b[6] != 0), "gated_unit: gradients of all weights or of none");
    return 0;
}
BTVAE_API long long btvae_gated_unit_bwd_bytes(const long long* unit, const long long* grads) {
    bk::Unit u;
    if (unit_of(unit, u) || check_back(u, grads)) return -1;
    bk::Pieces scratch = {nullptr, 0};
    bk::plan_backward(u, grads, scratch);
    return scratch.used;
}
BTVAE_API int btvae_gated_unit_bwd(const long long* unit, const long long* grads, const void* store, long long store_bytes, void* scratch, long long scratch_bytes, void* stream) {
    bk::Unit u;
    if (int rc = unit_of(unit, u)) return rc;
    if (int rc = check_back(u, grads)) return rc;
    const long long* b = grads;
    bk::Pieces kept = {(char*)const_cast<void*>(store), 0}, spare = {(char*)scratch, 0};
    const bk::Kept k = bk::lay_out(u, true, kept);
    const bk::BackwardPlan p = bk::plan_backward(u, b, spare);
    BTVAE_REQUIRE((store || u.M == 0) && kept.used <= store_bytes && scratch && spare.used <= scratch_bytes, "gated_unit: workspace too small");
    long long jobs[40];
    int n = 0;
    if (p.DY.pack) bk::add_job(jobs, n, (const void*)b[0], (int)b[1], b[2], p.DY.at, p.DY.ld, u.planes, u.M, u.N, bk::tiles(u.N, 32) * 32, 0);
    bk::add_job(jobs, n, u.wd, u.w16, u.ldd, p.WdT.at, p.WdT.ld, u.planes, u.N, u.F, p.WdT.width, 1);
    if (b[3]) {
        bk::add_job(jobs, n, u.wg, u.w16, u.ldg, p.WT.at, p.WT.ld, u.planes, u.F, u.K, p.half, 1);
        bk::add_job(jobs, n, u.wu, u.w16, u.ldu, (const char*)p.WT.at + bk::bytes_of(p.half, u.planes), p.WT.ld, u.planes, u.F, u.K, p.half, 1);
    }
    if (int rc = btvae_block_pack(jobs, n, stream)) return rc;
    if (int rc = btvae_gated_proj_bwd(p.DY.at, p.DY.ld, p.WdT.at, p.WdT.ld, k.kept, p.dGU, p.ldd, p.colpart, u.planes, u.act, u.M, u.F, p.DY.width, stream)) return rc;
    if (b[3])
        if (int rc = btvae_block_product(p.dGU, p.ldd, p.WT.at, p.WT.ld, nullptr, 0, (void*)b[3], u.K, u.x16, p.ws, p.dx_floats, u.planes, u.M, u.K, 2 * p.half, stream)) return rc;
    if (!b[4]) return 0;
    const int acc = b[14] != 0;
    const long long w[26] = {(long long)p.dGU, p.ldd, (long long)k.X.at, k.X.ld, b[4], u.F, b[5], p.half, u.F, u.K, b[10], 2 * p.half, u.K,
                             (long long)p.DY.at, p.DY.ld, (long long)k.H, k.ldh, b[6], u.N, 0, 0, 0, u.F, b[11], u.N, u.F};
    if (int rc = btvae_block_wgrad_pair(w, p.ws, p.w_floats, u.planes, u.M, acc, stream)) return rc;
    if (p.colpart)
        if (int rc = btvae_block_strip_sums(p.colpart, u.M ? btvae_gated_proj_strips(u.M) : 0, u.F, b[7] ? (void*)b[7] : p.other, (void*)b[8], (int)b[12], acc, stream)) return rc;
    if (b[9])
        if (int rc = btvae_block_colsum((const void*)b[0], (int)b[1], std::max<long long>(b[2], u.N), p.ws, p.c_floats, (void*)b[9], (int)b[13], acc, u.M, u.N, stream)) return rc;
    return 0;
}

// ---- few rows ----
BTVAE_API int btvae_few_rows_max(void) { return 32; }

template <int WT, bool GATED>
static int launch_few(const bk::FewArgs& p, bool vec, hipStream_t s, const char* what) {
    const dim3 grid((unsigned)bk::tiles(p.N, GATED ? 8 : 16));
    if (p.M <= 16) {
        if (vec) hipLaunchKernelGGL((bk::gemm_few<WT, GATED, 1, true>), grid, dim3(512), 0, s, p);
        else hipLaunchKernelGGL((bk::gemm_few<WT, GATED, 1, false>), grid, dim3(512), 0, s, p);
    } else {
        if (vec) hipLaunchKernelGGL((bk::gemm_few<WT, GATED, 2, true>), grid, dim3(512), 0, s, p);
        else hipLaunchKernelGGL((bk::gemm_few<WT, GATED, 2, false>), grid, dim3(512), 0, s, p);
    }
    return check_launch(what);
}
// Products with up to btvae_few_rows_max() rows; W2 null: C = X W^T + bias; else C = act(X W^T + bias) (X W2^T + bias2).  `w_bf16`: the
// weights and biases; X of their type, or (without W2) fp32; C of either.
BTVAE_API int btvae_few_rows(const void* X, int x_bf16, long long ldx, const void* W, const void* W2, int w_bf16, long long ldw, const void* bias, const void* bias2, void* C, int c_bf16, long long ldc,
                             int act, int M, int N, int K, void* stream) {
    BTVAE_REQUIRE(M >= 0 && M <= 32 && N > 0 && K > 0 && ldx >= K && ldw >= K && ldc >= N, "few_rows: bad sizes (M %d, N %d, K %d)", M, N, K);
    BTVAE_REQUIRE(act >= 0 && act <= 3, "few_rows: unknown activation %d", act);
    BTVAE_REQUIRE(!x_bf16 == !w_bf16 || (w_bf16 && !W2), "few_rows: unsupported pair of types");
    if (M == 0) return 0;
    bk::FewArgs p = {};
    const int sw = w_bf16 ? 2 : 4, gw = 16 / sw, gx = x_bf16 ? 8 : 4;
    p.X = X; p.ldx = ldx; p.x_bf16 = x_bf16; p.B = (const char*)W; p.B2 = (const char*)W2; p.ldb = ldw * sw;
    p.bias = bias; p.bias2 = bias2; p.bias_bf16 = w_bf16; p.C = C; p.ldc = ldc; p.c_bf16 = c_bf16; p.M = M; p.N = N; p.K = K; p.act = act;
    const bool vec = bk::al16(X) && bk::al16(W) && (!W2 || bk::al16(W2)) && K % gw == 0 && ldx % gx == 0 && ldw % gw == 0;
    hipStream_t s = BLK_STREAM(stream);
    ProfScope prof(PK_GEMM_FWD, s, (W2 ? 4.0 : 2.0) * M * N * K, 0.0);
    if (w_bf16 && !x_bf16) return launch_few<bk::W_BF16_X32, false>(p, vec, s, "few_rows");
    if (w_bf16) return W2 ? launch_few<bk::W_BF16, true>(p, vec, s, "few_rows") : launch_few<bk::W_BF16, false>(p, vec, s, "few_rows");
    return W2 ? launch_few<bk::W_F32, true>(p, vec, s, "few_rows") : launch_few<bk::W_F32, false>(p, vec, s, "few_rows");
}

// ---- 8-bit products ----
// q [rows][ldq] (ldq a multiple of 128), scale bytes e + 127 [rows][scp] (scp a multiple of 4), one for each 128 columns
BTVAE_API int btvae_fp8_quantize(const void* src, int src_bf16, long long ld, void* q, long long ldq, void* sc, long long scp, int rows, int K, void* stream) {
    const int kb = bk::tiles(K, 128);
    BTVAE_REQUIRE(rows >= 0 && K > 0 && ld >= K && ldq >= (long long)kb * 128 && (ldq & 15) == 0 && bk::al16(q) && scp >= kb, "fp8_quantize: bad layout");
    if (rows == 0) return 0;
    const unsigned grid = (unsigned)std::min<long long>(((long long)rows * kb + 15) / 16, 32768);
    hipStream_t s = BLK_STREAM(stream);
    if (src_bf16) hipLaunchKernelGGL((bk::quantize_rows<true>), dim3(grid), dim3(256), 0, s, src, ld, (unsigned char*)q, ldq, (unsigned char*)sc, scp, rows, K, kb);
    else hipLaunchKernelGGL((bk::quantize_rows<false>), dim3(grid), dim3(256), 0, s, src, ld, (unsigned char*)q, ldq, (unsigned char*)sc, scp, rows, K, kb);
    return check_launch("fp8_quantize");
}
// weights: one scale for each 128 x 128 block, scale bytes [ceil(N / 128)][scp]
BTVAE_API int btvae_fp8_quantize_blocks(const void* src, int src_bf16, long long ld, void* q, long long ldq, void* sc, long long scp, int N, int K, void* stream) {
    const int kb = bk::tiles(K, 128), nb = bk::tiles(N, 128);
    BTVAE_REQUIRE(N > 0 && K > 0 && ld >= K && ldq >= (long long)kb * 128 && (ldq & 15) == 0 && bk::al16(q) && scp >= kb && nb <= 65535, "fp8_quantize_blocks: bad layout");
    hipStream_t s = BLK_STREAM(stream);
    if (src_bf16) hipLaunchKernelGGL((bk::quantize_blocks<true>), dim3(kb, nb), dim3(256), 0, s, src, ld, (unsigned char*)q, ldq, (unsigned char*)sc, scp, N, K);
    else hipLaunchKernelGGL((bk::quantize_blocks<false>), dim3(kb, nb), dim3(256), 0, s, src, ld, (unsigned char*)q, ldq, (unsigned char*)sc, scp, N, K);
    return check_launch("fp8_quantize_blocks");
}
// out fp32 [rows][K]: the values that quantised rows (blocks = 0) or weights (blocks = 1) stand for
BTVAE_API int btvae_fp8_dequantize(const void* q, long long ldq, const void* sc, long long scp, int blocks, float* out, int rows, int K, void* stream) {
    BTVAE_REQUIRE(rows >= 0 && K > 0 && ldq >= K && scp >= bk::tiles(K, 128), "fp8_dequantize: bad layout");
    if (rows == 0) return 0;
    hipLaunchKernelGGL(bk::dequantize, dim3((unsigned)std::min<long long>(((long long)rows * K + 255) / 256, 16384)), dim3(256), 0, BLK_STREAM(stream), (const unsigned char*)q, ldq,
                       (const unsigned char*)sc, scp, blocks ? 7 : 0, out, rows, K);
    return check_launch("fp8_dequantize");
}

// out bf16 [rows][ldo]: the same values, exactly, zeros up to whole blocks of 128 columns
BTVAE_API int btvae_fp8_expand(const void* q, long long ldq, const void* sc, long long scp, int blocks, void* out, long long ldo, int rows, int K, void* stream) {
    const int kb = bk::tiles(K, 128);
    BTVAE_REQUIRE(rows >= 0 && K > 0 && ldq >= kb * 128LL && (ldq & 15) == 0 && bk::al16(q) && scp >= kb && ldo >= kb * 128LL && (ldo & 7) == 0 && bk::al16(out), "fp8_expand: bad layout");
    if (rows == 0) return 0;
    hipLaunchKernelGGL(bk::expand_rows, dim3((unsigned)std::min<long long>(((long long)rows * kb * 16 + 255) / 256, 16384)), dim3(256), 0, BLK_STREAM(stream), (const unsigned char*)q, ldq,
                       (const unsigned char*)sc, scp, blocks ? 7 : 0, (unsigned short*)out, ldo, rows, kb * 16);
    return check_launch("fp8_expand");
}

static bool fp8_ok(const void* q, long long ldq, const void* sc, long long scp, int K) {
    const int kb = bk::tiles(K, 128);
    return bk::al16(q) && (ldq & 15) == 0 && ldq >= (long long)kb * 128 && ((uintptr_t)sc & 3) == 0 && (scp & 3) == 0 && scp >= kb;
}
BTVAE_API long long btvae_fp8_product_ws(int M, int N, int K) {
    const bk::ProductPlan r = bk::plan_product(M, N, bk::tile_width(false), bk::tiles(K, 128), 4);
    return r.z > 1 ? (long long)r.z * M * N : 0;
}
BTVAE_API int btvae_fp8_product(const void* X, long long ldx, const void* xs, long long xsp, const void* W, long long ldw, const void* wsc, long long wscp, const float* bias,
                                void* C, long long ldc, int c_bf16, float* ws, long long ws_floats, int M, int N, int K, void* stream) {
    BTVAE_REQUIRE(M >= 0 && N > 0 && K > 0 && ldc >= N, "fp8_product: bad sizes (M %d, N %d, K %d)", M, N, K);
    if (M == 0) return 0;
    BTVAE_REQUIRE(fp8_ok(X, ldx, xs, xsp, K) && fp8_ok(W, ldw, wsc, wscp, K), "fp8_product: bad operand layout");
    hipStream_t s = BLK_STREAM(stream);
    bk::Args p = {};
    p.A = (const char*)X; p.lda = ldx; p.B = (const char*)W; p.ldb = ldw;
    p.M = M; p.N = N; p.K = K; p.ks = bk::tiles(K, 128);
    p.a_sc = (const unsigned char*)xs; p.a_scp = xsp; p.b_sc = (const unsigned*)wsc; p.b_scp = (int)(wscp / 4);
    const bk::ProductPlan r = bk::plan_product(M, N, bk::tile_width(false), p.ks, 4);
    BTVAE_REQUIRE(r.z == 1 || (ws && ws_floats >= (long long)r.z * M * N), "fp8_product: workspace too small");
    p.kz = r.kz; p.slab = ws; p.bias = bias;
    p.C = C; p.ldc = ldc; p.c_type = c_bf16 ? bk::T_BF16 : bk::T_F32;
    ProfScope prof(PK_GEMM_FWD, s, 2.0 * M * N * K, 0.0);
    if (int rc = bk::launch_rows<bk::FMT_E4M3, bk::EP_LINEAR>(p, r.z, s, "fp8_product")) return rc;
    if (r.z == 1) return 0;
    bk::SlabJobs q = {};
    q.n = 1;
    q.j[0] = {ws, r.z, M, N, C, ldc, M, nullptr, 0, 0, bias, 0, c_bf16, 0, 0, 0};
    return bk::launch_reduce(q, s, "fp8_product reduction");
}
// H = act(x Wg^T + bg) (x Wu^T + bu), quantised again (q [M][ldh], scale bytes [M][hsp]) in the epilogue.  expanded: X, Wg, Wu hold bf16 (pitches in
// elements, whole blocks of 128 columns) instead of e4m3 and scales.
BTVAE_API int btvae_fp8_gated_proj(const void* X, long long ldx, const void* xs, long long xsp, const void* Wg, const void* gs, const void* Wu, const void* us, long long ldw, long long wscp,
                                   int expanded, const float* bg, const float* bu, void* H, long long ldh, void* hs, long long hsp, int act, int M, int F, int K, void* stream) {
    BTVAE_REQUIRE(M >= 0 && F > 0 && K > 0, "fp8_gated_proj: bad sizes (M %d, F %d, K %d)", M, F, K);
    BTVAE_REQUIRE(act >= 0 && act <= 3, "fp8_gated_proj: unknown activation %d", act);
    if (M == 0) return 0;
    BTVAE_REQUIRE(fp8_ok(H, ldh, hs, hsp, F), "fp8_gated_proj: bad layout of H");
    bk::Args p = {};
    const int kp = bk::tiles(K, 128) * 128, sz = expanded ? 2 : 1;
    p.A = (const char*)X; p.lda = ldx * sz; p.B = (const char*)Wg; p.B2 = (const char*)Wu; p.ldb = ldw * sz;
    p.M = M; p.N = F;
    p.bias = bg; p.bias2 = bu; p.C = H; p.ldc = ldh; p.q_sc = (unsigned char*)hs; p.q_scp = hsp; p.act = act;
    ProfScope prof(PK_GEMM_FWD, BLK_STREAM(stream), 4.0 * M * F * K, 0.0);
    if (expanded) {
        BTVAE_REQUIRE(operand_ok(X, ldx * 2, 1, kp) && operand_ok(Wg, ldw * 2, 1, kp) && operand_ok(Wu, ldw * 2, 1, kp), "fp8_gated_proj: bad operand layout");
        p.K = kp; p.ks = p.kz = kp / 64;
        return bk::launch_rows<bk::FMT_BF16, bk::EP_GATED_Q>(p, 1, BLK_STREAM(stream), "fp8_gated_proj");
    }
    BTVAE_REQUIRE(fp8_ok(X, ldx, xs, xsp, K) && fp8_ok(Wg, ldw, gs, wscp, K) && fp8_ok(Wu, ldw, us, wscp, K), "fp8_gated_proj: bad operand layout");
    p.K = K; p.ks = p.kz = kp / 128;
    p.a_sc = (const unsigned char*)xs; p.a_scp = xsp; p.b_sc = (const unsigned*)gs; p.b2_sc = (const unsigned*)us; p.b_scp = (int)(wscp / 4);
    return bk::launch_rows<bk::FMT_E4M3, bk::EP_GATED_Q>(p, 1, BLK_STREAM(stream), "fp8_gated_proj");
}
// Up to btvae_few_rows_max() rows of fp32 / bf16 x, quantised on the way in; W2 null: C = x W^T + bias, else the gated product (C fp32 or bf16).
BTVAE_API int btvae_fp8_few_rows(const void* X, int x_bf16, long long ldx, const void* W, const void* wsc, const void* W2, const void* wsc2, long long ldw, long long wscp, const float* bias,
                                 const float* bias2, void* C, long long ldc, int c_bf16, int act, int M, int N, int K, void* stream) {
    BTVAE_REQUIRE(M >= 0 && M <= 32 && N > 0 && K > 0 && ldx >= K && ldc >= N, "fp8_few_rows: bad sizes (M %d, N %d, K %d)", M, N, K);
    BTVAE_REQUIRE(act >= 0 && act <= 3, "fp8_few_rows: unknown activation %d", act);
    BTVAE_REQUIRE(fp8_ok(W, ldw, wsc, wscp, K) && (!W2 || fp8_ok(W2, ldw, wsc2, wscp, K)), "fp8_few_rows: bad weight layout");
    if (M == 0) return 0;
    bk::FewArgs p = {};
    p.X = X; p.ldx = ldx; p.x_bf16 = x_bf16; p.B = (const char*)W; p.B2 = (const char*)W2; p.ldb = ldw;
    p.b_sc = (const unsigned char*)wsc; p.b2_sc = (const unsigned char*)wsc2; p.b_scp = wscp;
    p.bias = bias; p.bias2 = bias2; p.C = C; p.ldc = ldc; p.c_bf16 = c_bf16; p.M = M; p.N = N; p.K = K; p.act = act;
    const bool vec = bk::al16(X) && K % 8 == 0 && (ldx & (x_bf16 ? 7 : 3)) == 0;
    hipStream_t s = BLK_STREAM(stream);
    ProfScope prof(PK_GEMM_FWD, s, (W2 ? 4.0 : 2.0) * M * N * K, 0.0);
    return W2 ? launch_few<bk::W_E4M3, true>(p, vec, s, "fp8_few_rows") : launch_few<bk::W_E4M3, false>(p, vec, s, "fp8_few_rows");
}
