// Row norms around a residual block, fused with the block's gate, residual scale and addition.
//
//   u = post(y),  v = r + s g u,  n = pre(v)        post / pre: t / sqrt(mean t^2 + eps) w  or  (t - mean) / sqrt(var + eps) w + c
//
//   dv = d_stream + pre'(dn),  dg = s u dv (summed over the rows that share a gate row),  ds = sum_rows g u dv,
//   du = s g dv,  dy = post'(du);   norm'(d) = q (e - hat mean(e hat) [- mean(e)]),  e = d w,  q = 1 / deviation
//
// Memory bound: every matrix is read once and written once; a row stays in registers between its two norms.  Measured, bf16, 65,536 x 1000 with 4096
// gate rows: forward 117 us (4.6 TB/s), backward 182 (4.4 TB/s) and 11 for the column sums (a large copy: 5.1 TB/s); one row 3.6 us.  A row belongs to
// 1, 2, 4 or 8 waves (up to 512, 1024, 2048, 8192 columns), eight values to a lane (sixteen beyond 4096 columns); the two moments and every sum are fp32.  The next
// row is on its way while one is worked on.  Gate row of row r: r % G, the order of the framework's
// draws (draw s of profile b is row s B + b).  In the backward pass a group takes all (or one stretch) of the rows of one
// gate row, so that gate row's gradient is a running sum in registers; the gradients of the row weights are running
// sums too, joined over a workgroup's rows through LDS and over workgroups by a second launch, always in the same order.
#include "block_launch.h"
#include <algorithm>

using namespace btvae;
using btvae_block::f32x4; using btvae_block::u32x4; using btvae_block::pack2; using btvae_block::bf_lo; using btvae_block::bf_hi;
using btvae_block::bf_load; using btvae_block::bf_bits;

namespace btvae_norm {

enum { NONE = 0, RMS = 1, LAYER = 2 };

struct Args {
    const void* r; const void* y; const void* g; int G;       // residual, branch (null: none), gate [G, N] (null: none)
    float s; const float* sv;                                 // residual scale: a number, or [N]
    const float* w1; const float* c1; const float* w2; const float* c2;      // null: 1 / 0
    int post, pre; float eps;
    void* v; void* n;                                         // stream (null without a branch), normed (null: none)
    float* stats;                                             // [4][M]: mean, 1 / deviation of post, of pre (null: not kept)
    int M, N;
    // backward
    const void* dv; const void* dn;                           // upstream gradients (null: zero)
    void* dr; void* dy; void* dg;                             // null: not wanted; dg: [G, N], or fp32 parts when splits > 1
    float* dg_part;                                           // [splits][G][N]
    int splits, share;                                        // stretches a gate row's `share` rows are cut into
    float* part;                                              // [5][groups of workgroups][N]: dw1, dc1, dw2, dc2, ds
    int want;                                                 // bits of the five column sums wanted
};

template <bool H> __device__ __forceinline__ float ld1(const void* p, long long i) {
    return H ? bf_load(p, i) : reinterpret_cast<const float*>(p)[i];
}
template <bool H> __device__ __forceinline__ void st1(void* p, long long i, float v) {
    if (H) reinterpret_cast<unsigned short*>(p)[i] = bf_bits(v);
    else reinterpret_cast<float*>(p)[i] = v;
}

// A thread's 8 NV values of a row.  VEC: NV runs of 8 consecutive columns (N a multiple of 8, rows on 16 bytes); else column
// (8 j + e) T + t, whole lines to a wave whatever N is.  Columns past N read as zero.  `Raw` is what a row looks like on its way: the
// next row's loads are issued before the present row is worked on.
template <int T, int NV, bool VEC> struct Row {
    __device__ __forceinline__ static int col(int t, int j, int e) { return VEC ? (j * T + t) * 8 + e : (j * 8 + e) * T + t; }
    template <bool H> struct Raw { u32x4 v[NV][H ? 1 : 2]; };
    template <bool H> __device__ __forceinline__ static void fetch(const void* p, long long row0, int N, int t, Raw<H>& x) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (VEC) {
                const int c = col(t, j, 0);
                const u32x4* s = reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(p) + (row0 + min(c, N - 8)) * (H ? 2 : 4));
                x.v[j][0] = s[0];
                if constexpr (!H) x.v[j][1] = s[1];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const long long i = row0 + min(col(t, j, e), N - 1);
                    if constexpr (H) {
                        const unsigned u = reinterpret_cast<const unsigned short*>(p)[i];
                        x.v[j][0][e >> 1] = e & 1 ? x.v[j][0][e >> 1] | (u << 16) : u;
                    } else {
                        x.v[j][e >> 2][e & 3] = reinterpret_cast<const unsigned*>(p)[i];
                    }
                }
            }
        }
    }
    template <bool H> __device__ __forceinline__ static void unpack(const Raw<H>& x, int N, int t, float (&v)[8 * NV]) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = H ? (e & 1 ? bf_hi(x.v[j][0][e >> 1]) : bf_lo(x.v[j][0][e >> 1])) : __uint_as_float(x.v[j][H ? 0 : e >> 2][e & 3]);
                v[8 * j + e] = col(t, j, VEC ? 0 : e) < N ? f : 0.f;
            }
    }
    // bf16 rows leave past L2 in whole lines (8192 / 65,536 / 262,144 rows of 1000, forward and backward: 58 / 307 / 1212 us, through L2 60 / 326 / 1255; alone and
    // with a kernel that reads `normed` the forward pass gains as well); fp32 rows, two stores of 16 in 32 bytes a lane, gain nothing by it (65,536 rows 236 us forward, past L2 245)
    template <bool H> __device__ __forceinline__ static void store(void* p, long long row0, int N, int t, const float (&v)[8 * NV]) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (VEC) {
                const int c = col(t, j, 0);
                if (c >= N) continue;
                if (H) {
                    u32x4 q;
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[e] = pack2(v[8 * j + 2 * e], v[8 * j + 2 * e + 1]);
                    __builtin_nontemporal_store(q, reinterpret_cast<u32x4*>(reinterpret_cast<unsigned short*>(p) + row0 + c));
                } else {
                    float* d = reinterpret_cast<float*>(p) + row0 + c;
                    *reinterpret_cast<f32x4*>(d) = f32x4{v[8 * j], v[8 * j + 1], v[8 * j + 2], v[8 * j + 3]};
                    *reinterpret_cast<f32x4*>(d + 4) = f32x4{v[8 * j + 4], v[8 * j + 5], v[8 * j + 6], v[8 * j + 7]};
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int c = col(t, j, e);
                    if (c < N) st1<H>(p, row0 + c, v[8 * j + e]);
                }
            }
        }
    }
};

// A weight vector over the rows of a workgroup.  Rows of one wave share it in LDS (a wave then needs few enough registers for two
// to four waves a SIMD); longer rows, one to a workgroup, keep their part in registers.  Absent: a constant, zero past N.
template <int T, int NV, bool VEC> struct Vec {
    static constexpr bool LDS = T == 64;
    float reg[LDS ? 1 : 8 * NV];
    float* lds;
    bool present;
    float absent;
    __device__ __forceinline__ void init(const float* p, float other, int N, int t, float* room) {
        present = p != nullptr;
        absent = other;
        lds = room;
        if constexpr (LDS) {
            if (present)
                for (int i = threadIdx.x; i < 8 * NV * T; i += blockDim.x) lds[i] = i < N ? p[i] : 0.f;
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int c = Row<T, NV, VEC>::col(t, j, e);
                    reg[8 * j + e] = c < N ? (present ? p[c] : other) : 0.f;
                }
        }
    }
    __device__ __forceinline__ void get(int N, int t, float (&v)[8 * NV]) const {
        if constexpr (!LDS) {
#pragma unroll
            for (int i = 0; i < 8 * NV; ++i) v[i] = reg[i];
        } else if (present) {
            asm volatile("" ::: "memory");                    // read again for every row: kept over rows it would be registers after all
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if (VEC) {
                    const f32x4 a = *reinterpret_cast<const f32x4*>(lds + (j * T + t) * 8), b = *reinterpret_cast<const f32x4*>(lds + (j * T + t) * 8 + 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { v[8 * j + e] = a[e]; v[8 * j + 4 + e] = b[e]; }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[8 * j + e] = lds[(j * 8 + e) * T + t];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[8 * j + e] = Row<T, NV, VEC>::col(t, j, e) < N ? absent : 0.f;
        }
    }
};

// Sum over the T threads of a row.  One wave: lane exchanges; more: LDS, `red` of this row's waves, two slots used in turn so
// that one barrier a sum is enough.
template <int T> __device__ __forceinline__ float row_sum(float v, float* red, int& turn) {
    v = wave_sum(v);
    if constexpr (T > 64) {
        constexpr int W = T / 64;
        float* slot = red + turn * W;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) slot[(threadIdx.x >> 6) & (W - 1)] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) v += slot[i];
    }
    return v;
}

// mean (0 for RMS) and 1 / deviation of a row held in registers; columns past N hold zeros.  Layer norm takes the second
// moment about the mean, after the mean is known.
template <int T, int NV, bool VEC>
__device__ __forceinline__ void moments(const float (&x)[8 * NV], int kind, float eps, int N, int t, float* red, int& turn, float& mean, float& q) {
    mean = 0.f;
    if (kind == LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8 * NV; ++i) s += x[i];
        mean = row_sum<T>(s, red, turn) / (float)N;
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = Row<T, NV, VEC>::col(t, j, e) < N ? x[8 * j + e] - mean : 0.f;
            ss += d * d;
        }
    q = 1.f / sqrtf(row_sum<T>(ss, red, turn) / (float)N + eps);
}

template <bool RH, bool BH, int W, int NV, bool VEC>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void norm_fwd(const Args p) {
    constexpr int T = 64 * W, RPB = W == 1 ? 4 : 1, E = 8 * NV;
    typedef Row<T, NV, VEC> R;
    __shared__ float red[2 * W];
    __shared__ __attribute__((aligned(16))) float room[W == 1 ? 5 * 64 * E : 1];
    int turn = 0;
    const int t = threadIdx.x % T;
    Vec<T, NV, VEC> w1, c1, w2, c2, sv;
    w1.init(p.w1, 1.f, p.N, t, room);
    c1.init(p.c1, 0.f, p.N, t, room + 64 * E);
    sv.init(p.sv, p.s, p.N, t, room + 2 * 64 * E);
    w2.init(p.w2, 1.f, p.N, t, room + 3 * 64 * E);
    c2.init(p.c2, 0.f, p.N, t, room + 4 * 64 * E);
    if (W == 1) __syncthreads();
    typename R::template Raw<RH> rr;
    typename R::template Raw<BH> ry, rg;
    auto fetch = [&](int row) {
        const long long o = (long long)row * p.N;
        R::template fetch<RH>(p.r, o, p.N, t, rr);
        if (p.y) {
            R::template fetch<BH>(p.y, o, p.N, t, ry);
            if (p.g) R::template fetch<BH>(p.g, (long long)(row % p.G) * p.N, p.N, t, rg);
        }
    };
    int row = (int)blockIdx.x * RPB + threadIdx.x / T;
    if (row < p.M) fetch(row);
    for (; row < p.M; row += (int)gridDim.x * RPB) {
        const long long o = (long long)row * p.N;
        float v[E], x[E], f[E];
        R::template unpack<RH>(rr, p.N, t, v);
        float mean = 0.f, q = 1.f;
        if (p.y) {
            R::template unpack<BH>(ry, p.N, t, x);
            if (p.g) R::template unpack<BH>(rg, p.N, t, f);
            else {
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] = 1.f;
            }
        }
        if (row + (int)gridDim.x * RPB < p.M) fetch(row + (int)gridDim.x * RPB);
        if (p.y) {
            if (p.post != NONE) moments<T, NV, VEC>(x, p.post, p.eps, p.N, t, red, turn, mean, q);
            float w[E];
            sv.get(p.N, t, w);
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] *= w[i];         // scale times gate
            if (p.post != NONE) {
                w1.get(p.N, t, w);
#pragma unroll
                for (int i = 0; i < E; ++i) x[i] = (x[i] - mean) * q * w[i];
                if (p.c1) {
                    c1.get(p.N, t, w);
#pragma unroll
                    for (int i = 0; i < E; ++i) x[i] += w[i];
                }
            }
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] += f[i] * x[i];
            R::template store<RH>(p.v, o, p.N, t, v);
            if (p.stats && t == 0) { p.stats[row] = mean; p.stats[(long long)p.M + row] = q; }
        }
        if (p.n) {
            moments<T, NV, VEC>(v, p.pre, p.eps, p.N, t, red, turn, mean, q);
            float w[E];
            w2.get(p.N, t, w);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = (v[i] - mean) * q * w[i];
            if (p.c2) {
                c2.get(p.N, t, w);
#pragma unroll
                for (int i = 0; i < E; ++i) v[i] += w[i];
            }
            R::template store<BH>(p.n, o, p.N, t, v);
            if (p.stats && t == 0) { p.stats[2LL * p.M + row] = mean; p.stats[3LL * p.M + row] = q; }
        }
    }
}

// FULL: column sums of the biases and of the scale are wanted too.
template <bool RH, bool BH, int W, int NV, bool VEC, bool FULL>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void norm_bwd(const Args p) {
    constexpr int T = 64 * W, RPB = W == 1 ? 4 : 1, E = 8 * NV;
    typedef Row<T, NV, VEC> R;
    __shared__ float red[2 * W];
    __shared__ __attribute__((aligned(16))) float room[W == 1 ? 4 * 64 * E : 1];
    int turn = 0;
    const int t = threadIdx.x % T;
    const float inv_n = 1.f / (float)p.N;
    Vec<T, NV, VEC> w1, c1, w2, sv;
    w1.init(p.w1, 1.f, p.N, t, room);
    c1.init(p.c1, 0.f, p.N, t, room + 64 * E);
    sv.init(p.sv, p.s, p.N, t, room + 2 * 64 * E);
    w2.init(p.w2, 1.f, p.N, t, room + 3 * 64 * E);
    if (W == 1) __syncthreads();
    float aw1[E], aw2[E], ac1[FULL ? E : 1], ac2[FULL ? E : 1], as[FULL ? E : 1], dg[E];
#pragma unroll
    for (int i = 0; i < E; ++i) aw1[i] = aw2[i] = dg[i] = 0.f;
    if constexpr (FULL) {
#pragma unroll
        for (int i = 0; i < E; ++i) ac1[i] = ac2[i] = as[i] = 0.f;
    }
    // rows in the order this group takes them: the rows of a stretch of one gate row, then the next stretch
    const int units = p.G * p.splits;
    struct At { int unit, s, end, gr; };
    auto open = [&](int unit) {
        At a;
        a.unit = unit;
        const int split = unit / p.G;
        a.gr = unit - split * p.G;
        a.s = (int)((long long)p.share * split / p.splits);
        a.end = (int)((long long)p.share * (split + 1) / p.splits);
        return a;
    };
    typename R::template Raw<RH> rr, rd;
    typename R::template Raw<BH> ry, rn, rg;
    auto fetch = [&](const At& a) {
        const long long o = (long long)(a.s * p.G + a.gr) * p.N;
        if (p.y) R::template fetch<BH>(p.y, o, p.N, t, ry);
        if (p.dv) R::template fetch<RH>(p.dv, o, p.N, t, rd);
        if (p.dn) {
            R::template fetch<BH>(p.dn, o, p.N, t, rn);
            R::template fetch<RH>(p.r, o, p.N, t, rr);
        }
        if (p.y && p.g) R::template fetch<BH>(p.g, (long long)a.gr * p.N, p.N, t, rg);
    };
    At at = {0, 0, 0, 0};
    int unit = (int)blockIdx.x * RPB + threadIdx.x / T;
    const bool any = unit < units;                            // (every stretch has rows)
    if (any) {
        at = open(unit);
        fetch(at);
    }
    for (bool more = any; more;) {
        const int row = at.s * p.G + at.gr, gr = at.gr, split = at.unit / p.G;
        const long long o = (long long)row * p.N;
        float y[E], g[E], d[E], e[E], h[E], w[E];
        if (p.y) {
            R::template unpack<BH>(ry, p.N, t, y);
            if (p.g) R::template unpack<BH>(rg, p.N, t, g);
            else {
#pragma unroll
                for (int i = 0; i < E; ++i) g[i] = 1.f;
            }
        }
        if (p.dv) R::template unpack<RH>(rd, p.N, t, d);
        else {
#pragma unroll
            for (int i = 0; i < E; ++i) d[i] = 0.f;
        }
        if (p.dn) {
            R::template unpack<BH>(rn, p.N, t, e);
            R::template unpack<RH>(rr, p.N, t, h);
        }
        const float mean = p.post != NONE ? p.stats[row] : 0.f, q = p.post != NONE ? p.stats[(long long)p.M + row] : 1.f;
        const float mean2 = p.dn ? p.stats[2LL * p.M + row] : 0.f, q2 = p.dn ? p.stats[3LL * p.M + row] : 0.f;
        bool last = ++at.s == at.end;                         // of its stretch
        if (last) {
            const int next = at.unit + (int)gridDim.x * RPB;
            more = next < units;
            if (more) at = open(next);
        }
        if (more) fetch(at);
        if (p.y) {                                            // y becomes its normalised self, g scale times gate
            sv.get(p.N, t, w);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                y[i] = (y[i] - mean) * q;
                if constexpr (!FULL) g[i] *= w[i];
            }
        }
        auto branch = [&](float (&u)[E]) {                    // what the gate multiplies
            if (p.post == NONE) {
#pragma unroll
                for (int i = 0; i < E; ++i) u[i] = y[i];
                return;
            }
            w1.get(p.N, t, u);
#pragma unroll
            for (int i = 0; i < E; ++i) u[i] *= y[i];
            if (p.c1) {
                float c[E];
                c1.get(p.N, t, c);
#pragma unroll
                for (int i = 0; i < E; ++i) u[i] += c[i];
            }
        };
        if (p.dn) {
            // the stream as the forward pass had it before its rounding
            if (p.y) {
                float u[E];
                branch(u);
                if constexpr (FULL) sv.get(p.N, t, w);
#pragma unroll
                for (int i = 0; i < E; ++i) h[i] += (FULL ? w[i] * g[i] : g[i]) * u[i];
            }
            w2.get(p.N, t, w);
            float se = 0.f, seh = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                h[i] = (h[i] - mean2) * q2;                   // past N: finite, and met by e = 0 only
                aw2[i] += e[i] * h[i];
                if constexpr (FULL) ac2[i] += e[i];
                e[i] *= w[i];
                se += e[i];
                seh += e[i] * h[i];
            }
            seh = row_sum<T>(seh, red, turn) * inv_n;
            se = p.pre == LAYER ? row_sum<T>(se, red, turn) * inv_n : 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) d[i] += q2 * (e[i] - h[i] * seh - se);
        }
        if (p.dr) R::template store<RH>(p.dr, o, p.N, t, d);
        if (p.y) {
            float se = 0.f, seh = 0.f;
            branch(e);
            if constexpr (FULL) {
                sv.get(p.N, t, w);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float ud = e[i] * d[i];
                    dg[i] += w[i] * ud;
                    as[i] += g[i] * ud;
                    d[i] *= w[i] * g[i];
                }
            } else {
                sv.get(p.N, t, w);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    dg[i] += w[i] * (e[i] * d[i]);
                    d[i] *= g[i];
                }
            }
            if (p.post != NONE) {
                w1.get(p.N, t, w);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    aw1[i] += d[i] * y[i];
                    if constexpr (FULL) ac1[i] += d[i];
                    d[i] *= w[i];
                    se += d[i];
                    seh += d[i] * y[i];
                }
                seh = row_sum<T>(seh, red, turn) * inv_n;
                se = p.post == LAYER ? row_sum<T>(se, red, turn) * inv_n : 0.f;
#pragma unroll
                for (int i = 0; i < E; ++i) d[i] = q * (d[i] - y[i] * seh - se);
            }
            if (p.dy) R::template store<BH>(p.dy, o, p.N, t, d);
        }
        if (last) {
            if (p.y && p.g) {
                if (p.dg_part) R::template store<false>(p.dg_part, ((long long)split * p.G + gr) * p.N, p.N, t, dg);
                else if (p.dg) R::template store<BH>(p.dg, (long long)gr * p.N, p.N, t, dg);
            }
#pragma unroll
            for (int i = 0; i < E; ++i) dg[i] = 0.f;
        }
    }
    if (W == 1) __syncthreads();                              // the vectors' room becomes the meeting place of the rows' sums
    auto finish = [&](int k, auto& a) {
        if (!((p.want >> k) & 1)) return;                     // uniform
        if constexpr (W == 1) {
            const int wv = threadIdx.x >> 6;
            __syncthreads();
            if (wv > 0) {
#pragma unroll
                for (int i = 0; i < E; ++i) room[((wv - 1) * E + i) * 64 + t] = a[i];
            }
            __syncthreads();
            if (wv > 0) return;
#pragma unroll
            for (int i = 0; i < E; ++i) a[i] += (room[i * 64 + t] + room[(E + i) * 64 + t]) + room[(2 * E + i) * 64 + t];
        }
        R::template store<false>(p.part, ((long long)k * gridDim.x + blockIdx.x) * p.N, p.N, t, a);
    };
    finish(0, aw1);
    finish(2, aw2);
    if constexpr (FULL) {
        finish(1, ac1);
        finish(3, ac2);
        finish(4, as);
    }
}

struct FinishArgs { const float* part; int strips, N; float* out[5]; };
// out[k][n] = sum over workgroups of part[k][.][n]: 32 columns x 8 lanes of strips
__global__ __launch_bounds__(256) void norm_columns(const FinishArgs p) {
    __shared__ float red[8][33];
    float* out = p.out[blockIdx.y];
    if (!out) return;                                         // uniform
    const float* part = p.part + (long long)blockIdx.y * p.strips * p.N;
    const int c = (int)blockIdx.x * 32 + (threadIdx.x & 31), sl = threadIdx.x >> 5;
    float s = 0.f;
    if (c < p.N) {
#pragma unroll 8
        for (int r = sl; r < p.strips; r += 8) s += part[(long long)r * p.N + c];
    }
    red[sl][threadIdx.x & 31] = s;
    __syncthreads();
    if (sl != 0 || c >= p.N) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x & 31];
    out[c] = s;
}
// dg = sum over stretches
template <bool BH>
__global__ __launch_bounds__(256) void norm_gate_sum(const float* __restrict__ part, int splits, long long total, void* out) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        float s = 0.f;
        for (int k = 0; k < splits; ++k) s += part[(long long)k * total + i];
        st1<BH>(out, i, s);
    }
}

constexpr int MAX_N = 8192;
inline int waves_for(int N) { return N <= 512 ? 1 : N <= 1024 ? 2 : N <= 2048 ? 4 : 8; }

// workgroups of the backward pass (their column sums are joined by a second launch) and stretches of a gate row
struct BwdPlan { int groups, splits; };
static BwdPlan bwd_plan(int M, int N, int G) {
    const int W = waves_for(N), rpb = W == 1 ? 4 : 1;
    // row groups in flight: a few waves to a SIMD, fewer and each column sum is shorter.  Measured, us with the sums, at 512 / 768 / 1024 / 1366 / 2048 / 2732 groups:
    //   one wave a row: 500 columns bf16, 65,536 rows 513 / 393 / 271 / 274 / 158 / 163; 200 columns, 200,000 rows 838 / 628 / 425 / 325 / 222 / 230
    //   two: 1000 columns bf16, 65,536 rows of 4096 gate rows 320 / 252 / 190 / 176 / 216 / 184, 50,001 of 16,667 258 / 187 / 158 / 144 / 173 / 155,
    //     60,000 of 3000 299 / 213 / 174 / 189 / 156 / 173; fp32, no gate, 65,536 rows 535 / 400 / 326 / 451 / 435 / 379
    //   four: 1500 columns bf16, 65,536 rows 608 / 721 / 617 / 685 / 632 / 681; 2048 fp32, 32,768 rows 336 / 432 / 346 / 384 / 360 / 397
    //   eight (256 / 384 / 512 / 768): 4000 columns bf16, 16,384 rows 209 / 253 / 215 / 219; 8000 fp32, 10,000 rows 857 / 1038 / 863 / 890
    // What decides is how many of a kernel's workgroups a compute unit holds, which its types change: one number a width cannot suit all, and
    // those for four and eight waves lose a sixth to 512 and 256
    const int units = W == 1 ? 2048 : W == 2 ? 1366 : W == 4 ? 768 : 384;
    const int share = M / std::max(G, 1);
    BwdPlan b;
    b.splits = G >= units ? 1 : std::max(1, std::min(share, units / std::max(G, 1)));
    const long long work = (long long)G * b.splits;
    b.groups = (int)std::max(1LL, std::min<long long>((work + rpb - 1) / rpb, units / rpb));
    return b;
}

template <bool RH, bool BH, bool BWD>
static void launch(const Args& p, bool vec, int grid, hipStream_t s) {
    const int W = waves_for(p.N);
#define BTVAE_NORM_GO(WW, VV, XX) \
    do { if constexpr (BWD) { \
            if (p.want & 26) hipLaunchKernelGGL((norm_bwd<RH, BH, WW, VV, XX, true>), dim3(grid), dim3(WW == 1 ? 256 : 64 * WW), 0, s, p); \
            else hipLaunchKernelGGL((norm_bwd<RH, BH, WW, VV, XX, false>), dim3(grid), dim3(WW == 1 ? 256 : 64 * WW), 0, s, p); } \
         else hipLaunchKernelGGL((norm_fwd<RH, BH, WW, VV, XX>), dim3(grid), dim3(WW == 1 ? 256 : 64 * WW), 0, s, p); } while (0)
#define BTVAE_NORM_W(XX) do { if (W == 1) BTVAE_NORM_GO(1, 1, XX); else if (W == 2) BTVAE_NORM_GO(2, 1, XX); else if (W == 4) BTVAE_NORM_GO(4, 1, XX); \
        else if (p.N <= 4096) BTVAE_NORM_GO(8, 1, XX); else BTVAE_NORM_GO(8, 2, XX); } while (0)
    if (vec) BTVAE_NORM_W(true); else BTVAE_NORM_W(false);
#undef BTVAE_NORM_W
#undef BTVAE_NORM_GO
}

}  // namespace btvae_norm

namespace bn_ = btvae_norm;

static bool al(const void* q) { return ((uintptr_t)q & 15) == 0; }        // null counts as aligned

BTVAE_API int btvae_norm_max_columns(void) { return bn_::MAX_N; }

// types: bit 0 residual / stream are bf16 (else fp32), bit 1 branch / gate / normed are bf16; a bf16 residual needs a bf16 branch.
// post / pre: 0 none, 1 rms, 2 layer.
BTVAE_API int btvae_norm_gate_residual_fwd(const void* residual, const void* branch, const void* gate, int G, float scale, const float* scale_vec, const float* post_w, const float* post_b,
                                           const float* pre_w, const float* pre_b, int post, int pre, float eps, void* stream_out, void* normed, float* stats, int types, int M, int N, void* stream) {
    BTVAE_REQUIRE(M >= 0 && M <= btvae_block::MAX_ROWS, "norm_gate_residual: too many rows");
    BTVAE_REQUIRE(N > 0 && N <= bn_::MAX_N, "norm_gate_residual: %d columns (1 to %d)", N, bn_::MAX_N);
    BTVAE_REQUIRE(types == 0 || types == 2 || types == 3, "norm_gate_residual: a bf16 residual needs a bf16 branch");
    BTVAE_REQUIRE(post >= 0 && post <= 2 && pre >= 0 && pre <= 2 && eps >= 0.f, "norm_gate_residual: bad norm");
    if (M == 0) return 0;                                     // (empty matrices have no address to check)
    BTVAE_REQUIRE((branch != nullptr) == (stream_out != nullptr) && (pre != 0) == (normed != nullptr) && (branch || normed), "norm_gate_residual: outputs do not match what is asked for");
    BTVAE_REQUIRE(!gate || (branch && G > 0 && M % G == 0), "norm_gate_residual: %d rows are not a multiple of %d gate rows", M, G);
    bn_::Args p = {};
    p.r = residual; p.y = branch; p.g = gate; p.G = gate ? G : 1; p.s = scale; p.sv = scale_vec; p.w1 = post_w; p.c1 = post_b; p.w2 = pre_w; p.c2 = pre_b;
    p.post = post; p.pre = pre; p.eps = eps; p.v = stream_out; p.n = normed; p.stats = stats; p.M = M; p.N = N;
    const bool vec = N % 8 == 0 && al(residual) && al(branch) && al(gate) && al(stream_out) && al(normed);
    const int rpb = bn_::waves_for(N) == 1 ? 4 : 1;
    const int grid = (int)std::min<long long>(((long long)M + rpb - 1) / rpb, 2048);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    ProfScope prof(PK_BN, s, 0.0, (types == 3 ? 2.0 : 4.0) * M * N * 4);
    if (types == 0) bn_::launch<false, false, false>(p, vec, grid, s);
    else if (types == 2) bn_::launch<false, true, false>(p, vec, grid, s);
    else bn_::launch<true, true, false>(p, vec, grid, s);
    return check_launch("norm_gate_residual");
}

// floats of workspace: column sums of the workgroups, and the stretches of the gate's gradient
BTVAE_API long long btvae_norm_gate_residual_ws(int M, int N, int G) {
    if (M <= 0 || N <= 0 || N > bn_::MAX_N) return 0;
    const int g = G > 0 ? G : M;
    const bn_::BwdPlan b = bn_::bwd_plan(M, N, g);
    return 5LL * b.groups * N + (b.splits > 1 && G > 0 ? (long long)b.splits * g * N : 0);
}

// Gradients that are not wanted are null.  stats as the forward pass left them.
BTVAE_API int btvae_norm_gate_residual_bwd(const void* d_stream, const void* d_normed, const void* residual, const void* branch, const void* gate, int G, float scale, const float* scale_vec,
                                           const float* post_w, const float* post_b, const float* pre_w, int post, int pre, const float* stats, void* d_residual, void* d_branch, void* d_gate,
                                           float* d_scale, float* d_post_w, float* d_post_b, float* d_pre_w, float* d_pre_b, float* ws, long long ws_floats, int types, int M, int N, void* stream) {
    BTVAE_REQUIRE(M >= 0 && M <= btvae_block::MAX_ROWS, "norm_gate_residual_bwd: too many rows");
    BTVAE_REQUIRE(N > 0 && N <= bn_::MAX_N, "norm_gate_residual_bwd: %d columns (1 to %d)", N, bn_::MAX_N);
    BTVAE_REQUIRE(types == 0 || types == 2 || types == 3, "norm_gate_residual_bwd: a bf16 residual needs a bf16 branch");
    BTVAE_REQUIRE(post >= 0 && post <= 2 && pre >= 0 && pre <= 2, "norm_gate_residual_bwd: bad norm");
    BTVAE_REQUIRE(M == 0 || !d_normed || pre, "norm_gate_residual_bwd: a gradient of a norm that was not asked for");
    BTVAE_REQUIRE(!gate || M == 0 || (branch && G > 0 && M % G == 0), "norm_gate_residual_bwd: %d rows are not a multiple of %d gate rows", M, G);
    BTVAE_REQUIRE(M == 0 || (!d_branch && !d_gate && !d_scale && !d_post_w && !d_post_b) || branch, "norm_gate_residual_bwd: gradients of an absent branch");
    BTVAE_REQUIRE(!d_gate || (gate && G > 0), "norm_gate_residual_bwd: a gradient of an absent gate");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    bn_::Args p = {};
    const int g = gate && G > 0 ? G : std::max(M, 1);
    const bn_::BwdPlan b = bn_::bwd_plan(std::max(M, 1), N, g);
    const long long parts = 5LL * b.groups * N, gp = b.splits > 1 && gate ? (long long)b.splits * g * N : 0;
    BTVAE_REQUIRE(M == 0 || (ws && ws_floats >= parts + gp), "norm_gate_residual_bwd: workspace too small");
    bn_::FinishArgs f = {};
    f.part = ws; f.strips = M == 0 ? 0 : b.groups; f.N = N;
    f.out[0] = d_post_w; f.out[1] = d_post_b; f.out[2] = d_normed || M == 0 ? d_pre_w : nullptr; f.out[3] = d_normed || M == 0 ? d_pre_b : nullptr; f.out[4] = d_scale;
    p.y = branch; p.g = gate; p.G = g; p.s = scale; p.sv = scale_vec; p.w1 = post_w; p.c1 = post_b; p.w2 = pre_w; p.post = post; p.pre = pre;
    p.r = residual; p.stats = const_cast<float*>(stats); p.M = M; p.N = N;
    p.dv = d_stream; p.dn = d_normed; p.dr = d_residual; p.dy = d_branch; p.dg = d_gate; p.dg_part = gp ? ws + parts : nullptr;
    p.splits = b.splits; p.share = M / g; p.part = ws;
    for (int k = 0; k < 5; ++k) p.want |= f.out[k] ? 1 << k : 0;
    if (M > 0) {
        const bool vec = N % 8 == 0 && al(d_stream) && al(d_normed) && al(residual) && al(branch) && al(gate) && al(d_residual) && al(d_branch) && al(d_gate) && (!p.dg_part || al(p.dg_part)) && al(ws);
        ProfScope prof(PK_BN, s, 0.0, (types == 3 ? 2.0 : 4.0) * M * N * 6);
        if (types == 0) bn_::launch<false, false, true>(p, vec, b.groups, s);
        else if (types == 2) bn_::launch<false, true, true>(p, vec, b.groups, s);
        else bn_::launch<true, true, true>(p, vec, b.groups, s);
        if (int rc = check_launch("norm_gate_residual_bwd")) return rc;
    }
    if (d_gate && (gp || M == 0)) {                           // (no rows: G x N sums of nothing)
        const long long total = (long long)(M == 0 ? G : g) * N;
        const int splits = M == 0 ? 0 : b.splits;
        const unsigned grid = (unsigned)std::min<long long>((total + 255) / 256, 8192);
        if (types & 2) hipLaunchKernelGGL((bn_::norm_gate_sum<true>), dim3(grid), dim3(256), 0, s, (const float*)p.dg_part, splits, total, d_gate);
        else hipLaunchKernelGGL((bn_::norm_gate_sum<false>), dim3(grid), dim3(256), 0, s, (const float*)p.dg_part, splits, total, d_gate);
        if (int rc = check_launch("norm_gate_residual_bwd gate")) return rc;
    }
    if (p.want) {
        hipLaunchKernelGGL(bn_::norm_columns, dim3((unsigned)((N + 31) / 32), 5), dim3(256), 0, s, f);
        return check_launch("norm_gate_residual_bwd columns");
    }
    return 0;
}
