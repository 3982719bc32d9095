// nnsp_delta_chunk.h -- the gated delta rule over chunks of 64 frames on the
// matrix cores (include/nnsp_seq.h); one .hip file per element type launches it.
//
// Within a chunk, with G_i the sum of g up to frame i and S0 the state before it,
//
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j   (j < i)        T = (I + A)^-1
//   U    = T (beta V - beta e^G (K S0))
//   O    = scale (e^G (Q S0) + P U)         P_ij = e^(G_i - G_j) q_i . k_j (j <= i)
//   S1   = e^(G_63) S0 + K^T (e^(G_63 - G) U)
//
// which is the rule of 64 frames with the recurrence left in one 64 x 64
// triangular inverse.  T and P need no state; the rest is five matrix products.
//
// Numbers.  The state, T and U are 32-bit values, and the matrix cores take 16
// bits: each is scaled by a power of two (its column's or row's largest to
// 2^14 .. 2^15) and split into an fp16 high and low part, 22 bits in all, and
// products keep hi hi + hi lo + lo hi, accumulated in 32 bits.  Rows of q and k
// are scaled the same way, which makes one fp16 part exact for bf16 and fp16
// (bf16 to 2^-39 of the row's largest); fp32 takes two.  All other factors
// (norms, decays, beta) multiply in 32 bits outside the products.  For bf16
// outputs the products that reach only the output (Q S0, P U) use one part of
// S0, P and U, 11 bits, below the output's own 8.
//
// Layout.  A wave owns 16 NB columns of the state and keeps them in registers
// in the 16x16 accumulator layout (lane: column lane % 16, rows 4 (lane / 16)
// .. + 3).  The k index of an MFMA is any order both operands agree on, so two
// accumulator tiles are, split to fp16, the B operand of a 32-deep product as
// they stand: K S0 -> R -> U -> S1 never leaves the registers, and only the A
// operands, which all waves share, come from LDS.
#ifndef NNSP_DELTA_CHUNK_H
#define NNSP_DELTA_CHUNK_H
#include <type_traits>

#include "nnsp_seq_dev.h"
#include "nnsp_seqk.h"

namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr int C = 64;       // frames of a chunk

__device__ __forceinline__ f32x4 mma(h8 a, h8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// power of two that takes m's magnitude to [2^14, 2^15), and its inverse
__device__ __forceinline__ float scale_of(float m, float& inv) {
    const int e = (__float_as_int(m) >> 23) & 255;
    const int s = min(max(268 - e, 1), 253);
    inv = __int_as_float((254 - s) << 23);
    return __int_as_float(s << 23);
}
__device__ __forceinline__ float max_xor16_32(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
template <int CTRL>
__device__ __forceinline__ float max_dpp(float x) {
    return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true)));
}
// largest over the 16 lanes of a row
__device__ __forceinline__ float max_row16(float x) {
    return max_dpp<0x128>(max_dpp<0x141>(max_dpp<0x4e>(max_dpp<0xb1>(x))));
}
__device__ __forceinline__ float amax4(float m, const f32x4& x) {
    return fmaxf(fmaxf(fmaxf(m, fabsf(x[0])), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
}

// keeps the operands of later products out of the registers until theirs are done
__device__ __forceinline__ void no_hoist() { __builtin_amdgcn_sched_barrier(0); }

// a copy the compiler knows nothing about: LDS addresses made of it are not
// kept in registers from chunk to chunk
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// two accumulator tiles times s as the high and low B operand of a 32-deep product
__device__ __forceinline__ void split(const f32x4& a, const f32x4& b, float s, h8& hi, h8& lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = i < 4 ? a[i & 3] : b[i & 3];
        hi[i] = (_Float16)(x * s);
        lo[i] = (_Float16)fmaf(x, s, -(float)hi[i]);
    }
}
__device__ __forceinline__ h8 high(const f32x4& a, const f32x4& b, float s) {
    h8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)((i < 4 ? a[i & 3] : b[i & 3]) * s);
    return r;
}

// 4 rows x 4 columns per lane group, transposed: lane l of 16 gets column l of rows 0 .. 3
__device__ __forceinline__ s4 read_tr(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
}

// T and P in LDS: row tiles 0 and 1 hold 32 frames a row, 2 and 3 all 64, in the
// k order of two stacked accumulator tiles; 8 halves of padding spread 16 rows
// over all banks
struct Tri {
    alignas(16) _Float16 x[32 * 40 + 32 * 72];
    // frames 32 s + 8-element group g of row
    __device__ __forceinline__ h8 operand(int m, int l15, int s, int g) const {
        return *reinterpret_cast<const h8*>(x + (m < 2 ? (16 * m + l15) * 40 : 1280 + (16 * m - 32 + l15) * 72) + 32 * s + 8 * g);
    }
    // frames 16 j + 4 g .. + 3 of row 16 m + l15
    __device__ __forceinline__ void put(int m, int l15, int j, int g, h4 v) {
        *reinterpret_cast<h4*>(x + (m < 2 ? (16 * m + l15) * 40 : 1280 + (16 * m - 32 + l15) * 72) + 32 * (j >> 1) + 8 * g + 4 * (j & 1)) = v;
    }
};

template <class T, int NKT, int NB>
struct Geo {
    static constexpr bool WIDE = std::is_same<T, float>::value;       // 32-bit input
    static constexpr int KP = WIDE ? 2 : 1;                           // parts of q and k
    static constexpr int OP = std::is_same<T, __bf16>::value ? 1 : 2; // parts of what only the output takes
    static constexpr int KS = NKT * 32 + 8;                           // row of K and Q, halves
    static constexpr int W = 64 * NB;                                 // columns of a workgroup
    static constexpr int VS = 16 * NB + (WIDE ? 4 : 8);               // row of a wave's V, elements
};

template <class T, int NKT, int NB>
struct Lds {
    using G = Geo<T, NKT, NB>;
    alignas(16) _Float16 K[G::KP][C][G::KS], Q[G::KP][C][G::KS];
    union {
        Tri T_[2];
        float D[4][16][20];        // transposed inverses of the diagonal blocks, until T is written
    };
    Tri P_[G::OP];
    union {
        alignas(16) float A[C][C + 4];  // A transposed, until T is done
        alignas(16) T V[4][C][G::VS];   // from then on: each wave's columns of v, then of out
    };
    // factors of a frame; e() is a decay, G the sum of g, s and e the first and last frame of its 16
    alignas(16) float kx[C], qx[C], kn[C], qn[C];  // norm times 2^-scale, length after the norm
    alignas(16) float gh[C], gl[C], beta[C];       // log2 of the decay up to the frame (two parts), beta
    alignas(16) float ab[C], ar[C];                // A rows: beta kx, times e(G - G_s)
    alignas(16) float pb[C], pr[C], pi[C];         // P rows: qx 2^scale, times e(G - G_s); 2^-scale
    alignas(16) float kc[C];                       // columns of both: kx e(G_e - G)
    alignas(16) float fx[C], fk[C], fq[C];         // of K S0, of U into the state, of Q S0
    float ti[4];                                   // 2^-scale of T's row tiles
    float all;                                     // decay over the whole chunk
};

// raw rows of q and k on their way to LDS: thread (row, quarter) holds chunks of
// 8 elements quarter, quarter + 4, ...
template <class T, int NKT>
struct RawRows {
    typename Vec<T, 8>::raw x[NKT];
};
template <class T, int NKT, bool FAST>
__device__ __forceinline__ void fetch_rows(RawRows<T, NKT>& r, const T* p, int quarter, int n, bool live) {
#pragma unroll
    for (int i = 0; i < NKT; ++i) {
        const int c = (quarter + 4 * i) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) r.x[i][j] = (T)0.0f;
        if (FAST) {
            if (live && c < n) r.x[i] = *reinterpret_cast<const typename Vec<T, 8>::type*>(p + 32 * i);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (live && c + j < n) r.x[i][j] = p[32 * i + j];
        }
    }
}
// scaled fp16 parts to LDS; returns 2^-scale, sets the sum of squares
template <class T, int NKT, int KP, int KS>
__device__ __forceinline__ float stage_rows(const RawRows<T, NKT>& r, _Float16 (*dst)[C][KS], int row, int quarter, float& ss) {
    float m = 0.0f;
    ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NKT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = (float)r.x[i][j];
            m = fmaxf(m, fabsf(x));
            ss = fmaf(x, x, ss);
        }
    m = max_dpp<0x4e>(max_dpp<0xb1>(m));
    ss = add_xor2(add_xor1(ss));
    float inv;
    const float s = scale_of(m, inv);
#pragma unroll
    for (int i = 0; i < NKT; ++i) {
        h8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = (float)r.x[i][j];
            hi[j] = (_Float16)(x * s);
            if (KP == 2) lo[j] = (_Float16)fmaf(x, s, -(float)hi[j]);
        }
        const int c = (quarter + 4 * i) * 8;
        *reinterpret_cast<h8*>(&dst[0][row][c]) = hi;
        if (KP == 2) *reinterpret_cast<h8*>(&dst[KP - 1][row][c]) = lo;
    }
    return inv;
}

// tile (mi, mj) of X Y^T
template <int NKT, int KP, int KS>
__device__ __forceinline__ f32x4 dot_tile(const _Float16 (*X)[C][KS], const _Float16 (*Y)[C][KS], int mi, int mj, int l15, int g) {
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < NKT; ++s) {
        const int c = 32 * s + 8 * g;
        const h8 a = *reinterpret_cast<const h8*>(&X[0][16 * mi + l15][c]), b = *reinterpret_cast<const h8*>(&Y[0][16 * mj + l15][c]);
        acc = mma(a, b, acc);
        if (KP == 2) {
            const h8 al = *reinterpret_cast<const h8*>(&X[KP - 1][16 * mi + l15][c]);
            const h8 bl = *reinterpret_cast<const h8*>(&Y[KP - 1][16 * mj + l15][c]);
            acc = mma(a, bl, mma(al, b, acc));
        }
    }
    return acc;
}
__device__ __forceinline__ f32x4 ld4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }

// Everything of the staged chunk that needs no state, by all four waves: the
// factors, T and P.  Starts and ends with the workgroup together.
//
// A decay between two frames of different 16s is a product of three that are
// each at most 1 (to the end of the column's 16, between, from the start of
// the row's), so it costs two multiplications an element; within a 16 it is an
// exponential of the difference.  P's row scale comes from a bound (lengths of
// q and k, the largest decay ratio), which an fp16's exponent has room for.
template <class T, int NKT, int NB>
__device__ __forceinline__ void make_tp(Lds<T, NKT, NB>& L, int wave, int lane, int nt) {
    using G = Geo<T, NKT, NB>;
    const int l15 = lane & 15, g = lane >> 4;
    f32x4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j <= wave) acc[j] = dot_tile<NKT, G::KP, G::KS>(L.K, L.K, wave, j, l15, g);
    {
        const int i = lane, s = i & ~15, e = i | 15;
        const float h = L.gh[i], l = L.gl[i], kx = L.kx[i];
        if (wave == 0) {
            const float b = L.beta[i] * kx, r = exp2_fast((h - L.gh[s]) + (l - L.gl[s]));
            L.ab[i] = b;
            L.ar[i] = b * r;
            L.kc[i] = exp2_fast((L.gh[e] - h) + (L.gl[e] - l)) * kx;
        } else if (wave == 1) {
            // largest decay ratio of a row: e(G_i - min over j <= i of G_j); largest length of a key
            float lo = h, kn = L.kn[i];
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const float y = __shfl_up(lo, d);
                if (lane >= d) lo = fminf(lo, y);
                kn = fmaxf(kn, __shfl_xor(kn, d));
            }
            float inv;
            const float qx = L.qx[i], sc = scale_of(L.qn[i] * kn * exp2_fast(fminf(h - lo, 120.0f)), inv);
            L.pi[i] = inv;
            L.pb[i] = qx * sc;
            L.pr[i] = qx * sc * exp2_fast((h - L.gh[s]) + (l - L.gl[s]));
        } else if (wave == 2) {
            const float up = exp2_fast(h);
            L.fx[i] = L.beta[i] * up * kx;
            L.fq[i] = up * L.qx[i];
            L.fk[i] = exp2_fast((L.gh[C - 1] - h) + (L.gl[C - 1] - l)) * kx;
            if (i == C - 1) L.all = up;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j > wave) continue;
        const int col = 16 * j + l15, row = 16 * wave + 4 * g;
        f32x4 f;
        if (j == wave) {
            const f32x4 h = ld4(&L.gh[row]), l = ld4(&L.gl[row]), b = ld4(&L.ab[row]);
            const float hj = L.gh[col], lj = L.gl[col], kj = L.kx[col];
#pragma unroll
            for (int r = 0; r < 4; ++r) f[r] = exp2_fast(fminf((h[r] - hj) + (l[r] - lj), 120.0f)) * (b[r] * kj);
        } else {
            const float k = L.kc[col] * exp2_fast(L.gh[16 * wave] - L.gh[16 * j + 15]);
            f = ld4(&L.ar[row]) * k;
        }
        *reinterpret_cast<f32x4*>(&L.A[col][row]) = acc[j] * f;
    }
    __syncthreads();
    if (wave == 0) {
        // the four diagonal blocks, a column of the inverse per lane, by substitution from the top
        const int b = 16 * g;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = i == l15 ? 1.0f : 0.0f;
#pragma unroll
        for (int j = 0; j < 15; ++j) {
#pragma unroll
            for (int q = (j + 1) / 4; q < 4; ++q) {
                const f32x4 a = ld4(&L.A[b + j][b + 4 * q]);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (4 * q + r > j) x[4 * q + r] = fmaf(-a[r], x[j], x[4 * q + r]);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) *reinterpret_cast<f32x4*>(&L.D[g][l15][4 * q]) = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
    } else {
        // P meanwhile: rows of tile 3, 2, and 1 with 0; as K Q^T, so that a lane has 4 frames of a row
        const int first = wave == 1 ? 3 : wave == 2 ? 2 : 0, last = wave == 3 ? 1 : first;
        for (int mi = first; mi <= last && mi < nt; ++mi) {
            const int row = 16 * mi + l15;
            const float pb = L.pb[row], pr = L.pr[row], hi_ = L.gh[row], li = L.gl[row], hs = L.gh[16 * mi];
            for (int j = 0; j <= (mi | 1); ++j) {
                h4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
                if (j <= mi) {
                    const f32x4 p = dot_tile<NKT, G::KP, G::KS>(L.K, L.Q, j, mi, l15, g);
                    const int col = 16 * j + 4 * g;
                    f32x4 f;
                    if (j == mi) {
                        const f32x4 h = ld4(&L.gh[col]), l = ld4(&L.gl[col]), k = ld4(&L.kx[col]);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            f[r] = col + r <= row ? exp2_fast(fminf((hi_ - h[r]) + (li - l[r]), 120.0f)) * (k[r] * pb) : 0.0f;
                    } else {
                        f = ld4(&L.kc[col]) * (pr * exp2_fast(hs - L.gh[16 * j + 15]));
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = j == mi && col + r > row ? 0.0f : p[r] * f[r];
                        a[r] = (_Float16)x;
                        b[r] = (_Float16)(x - (float)a[r]);
                    }
                }
                L.P_[0].put(mi, l15, j, g, a);
                if (G::OP == 2) L.P_[G::OP - 1].put(mi, l15, j, g, b);
            }
        }
    }
    __syncthreads();
    // block row i = wave of T, transposed: N_ij = -T_jj^T sum over j < k <= i of A_kj^T N_ik, in 32 bits
    f32x4 t[4];
    float m = 0.0f;
#pragma unroll
    for (int j = 3; j >= 0; --j) {
        t[j] = f32x4{0, 0, 0, 0};
        if (j > wave || wave >= nt) continue;
        if (j == wave) {
#pragma unroll
            for (int r = 0; r < 4; ++r) t[j][r] = L.D[j][4 * g + r][l15];
        } else {
            f32x4 y = {0, 0, 0, 0};
#pragma unroll
            for (int k = j + 1; k < 4; ++k) {
                if (k > wave) continue;
                const f32x4 a = ld4(&L.A[16 * j + l15][16 * k + 4 * g]);
#pragma unroll
                for (int r = 0; r < 4; ++r) y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], t[k][r], y, 0, 0, 0);
            }
            const f32x4 d = ld4(&L.D[j][l15][4 * g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) t[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(-d[r], y[r], t[j], 0, 0, 0);
        }
        m = amax4(m, t[j]);
    }
    __syncthreads();
    if (wave < nt) {
        float inv;
        const float s = scale_of(max_xor16_32(max_row16(m)), inv);
        if (lane == 0) L.ti[wave] = inv;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > (wave | 1)) continue;
            h4 a, b;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                a[r] = (_Float16)(t[j][r] * s);
                b[r] = (_Float16)fmaf(t[j][r], s, -(float)a[r]);
            }
            L.T_[0].put(wave, l15, j, g, a);
            L.T_[1].put(wave, l15, j, g, b);
        }
    }
    __syncthreads();
}

// The products with the state for one chunk of nt live tiles of 16 frames: this
// wave's columns.  S holds the state times 1 / sinv (a power of two per column);
// between() runs once the state's 16-bit parts are dead (it holds the next
// chunk's loads).
template <class T, int NKT, int NB, class F>
__device__ __forceinline__ void advance(Lds<T, NKT, NB>& L, f32x4 (&S)[2 * NKT][NB], float (&sinv)[NB], int wave, int lane,
                                        int nt, const F& between) {
    using G = Geo<T, NKT, NB>;
    const int l15 = lane & 15, g = lane >> 4;
    f32x4 R[4][NB], O[4][NB];
    float smax[NB];
    {
        h8 hi[NKT][NB], lo[NKT][NB];
        float inv[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float m = 0.0f;
#pragma unroll
            for (int t = 0; t < 2 * NKT; ++t) m = amax4(m, S[t][n]);
            smax[n] = max_xor16_32(m);
            const float s = scale_of(smax[n], inv[n]);
            inv[n] *= sinv[n];
#pragma unroll
            for (int t = 0; t < NKT; ++t) split(S[2 * t][n], S[2 * t + 1][n], s, hi[t][n], lo[t][n]);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            f32x4 x[NB], o[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) R[m][n] = O[m][n] = x[n] = o[n] = f32x4{0, 0, 0, 0};
            if (m >= nt) continue;
            no_hoist();
#pragma unroll
            for (int s = 0; s < NKT; ++s) {
                const int c = 32 * s + 8 * g;
                const h8 k = *reinterpret_cast<const h8*>(&L.K[0][16 * m + l15][c]);
                const h8 q = *reinterpret_cast<const h8*>(&L.Q[0][16 * m + l15][c]);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    x[n] = mma(k, lo[s][n], mma(k, hi[s][n], x[n]));
                    o[n] = mma(q, hi[s][n], o[n]);
                    if (G::OP == 2) o[n] = mma(q, lo[s][n], o[n]);
                }
                if (G::KP == 2) {
                    const h8 kl = *reinterpret_cast<const h8*>(&L.K[G::KP - 1][16 * m + l15][c]);
                    const h8 ql = *reinterpret_cast<const h8*>(&L.Q[G::KP - 1][16 * m + l15][c]);
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        x[n] = mma(kl, hi[s][n], x[n]);
                        o[n] = mma(ql, hi[s][n], o[n]);
                    }
                }
            }
            const f32x4 b = ld4(&L.beta[16 * m + 4 * g]), fx = ld4(&L.fx[16 * m + 4 * g]), fq = ld4(&L.fq[16 * m + 4 * g]);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float v[4];
                if constexpr (G::WIDE) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = L.V[wave][16 * m + 4 * g + r][16 * n + l15];
                } else {
                    const auto t = __builtin_bit_cast(typename Vec<T, 4>::raw,
                                                      read_tr(&L.V[wave][16 * m + 4 * g + (l15 >> 2)][16 * n + 4 * (l15 & 3)]));
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = (float)t[r];
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    R[m][n][r] = fmaf(-fx[r] * inv[n], x[n][r], b[r] * v[r]);
                    O[m][n][r] = fq[r] * inv[n] * o[n][r];
                }
            }
        }
    }
    between();
    f32x4 U[4][NB];
    {
        h8 hi[2][NB], lo[2][NB];
        float inv[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float m = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t) m = amax4(m, R[t][n]);
            const float s = scale_of(max_xor16_32(m), inv[n]);
#pragma unroll
            for (int t = 0; t < 2; ++t) split(R[2 * t][n], R[2 * t + 1][n], s, hi[t][n], lo[t][n]);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            f32x4 u[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) U[m][n] = u[n] = f32x4{0, 0, 0, 0};
            if (m >= nt) continue;
            no_hoist();
#pragma unroll
            for (int s = 0; s <= m / 2; ++s) {
                const h8 th = L.T_[0].operand(m, l15, s, g), tl = L.T_[1].operand(m, l15, s, g);
#pragma unroll
                for (int n = 0; n < NB; ++n) u[n] = mma(tl, hi[s][n], mma(th, lo[s][n], mma(th, hi[s][n], u[n])));
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) U[m][n] = u[n] * (L.ti[m] * inv[n]);
        }
    }
    // O += P U
    {
        h8 hi[2][NB], lo[2][NB];
        float inv[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float m = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t) m = amax4(m, U[t][n]);
            const float s = scale_of(max_xor16_32(m), inv[n]);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (G::OP == 2) split(U[2 * t][n], U[2 * t + 1][n], s, hi[t][n], lo[t][n]);
                else hi[t][n] = high(U[2 * t][n], U[2 * t + 1][n], s);
            }
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            if (m >= nt) continue;
            no_hoist();
            f32x4 o[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) o[n] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s <= m / 2; ++s) {
                const h8 ph = L.P_[0].operand(m, l15, s, g);
#pragma unroll
                for (int n = 0; n < NB; ++n) o[n] = mma(ph, hi[s][n], o[n]);
                if (G::OP == 2) {
                    const h8 pl = L.P_[G::OP - 1].operand(m, l15, s, g);
#pragma unroll
                    for (int n = 0; n < NB; ++n) o[n] = mma(pl, hi[s][n], mma(ph, lo[s][n], o[n]));
                }
            }
            const f32x4 pi = ld4(&L.pi[16 * m + 4 * g]);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    L.V[wave][16 * m + 4 * g + r][16 * n + l15] = (T)fmaf(o[n][r], pi[r] * inv[n], O[m][n][r]);
        }
    }
    // S1, accumulated onto the decayed state in U's scale; where U is next to nothing, in 2^13 of the decayed state's
    // own, so that neither leaves its range (2^100 at most: the state's factor f stays finite)
    {
        h8 hi[2][NB], lo[2][NB];
        const float all = L.all;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float m = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                U[t][n] *= ld4(&L.fk[16 * t + 4 * g]);
                m = amax4(m, U[t][n]);
            }
            float inv;
            const float s = scale_of(fmaxf(fmaxf(max_xor16_32(m), smax[n] * sinv[n] * (all * 0x1p-13f)), 0x1p-86f), inv);
#pragma unroll
            for (int t = 0; t < 2; ++t) split(U[2 * t][n], U[2 * t + 1][n], s, hi[t][n], lo[t][n]);
            const float f = all * s * sinv[n];
#pragma unroll
            for (int t = 0; t < 2 * NKT; ++t) S[t][n] *= f;
            sinv[n] = inv;
        }
#pragma unroll
        for (int t = 0; t < 2 * NKT; ++t) {
            if (t & 1) no_hoist();
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (2 * s >= nt) continue;
                const int row = 32 * s + 4 * g + (l15 >> 2), col = 32 * (t >> 1) + 8 * (l15 & 3) + 4 * (t & 1);
                const auto kt = [&](int part) {
                    const s4 a = read_tr(&L.K[part][row][col]), b = read_tr(&L.K[part][row + 16][col]);
                    const h4 x = __builtin_bit_cast(h4, a), y = __builtin_bit_cast(h4, b);
                    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                };
                const h8 k = kt(0);
#pragma unroll
                for (int n = 0; n < NB; ++n) S[t][n] = mma(k, lo[s][n], mma(k, hi[s][n], S[t][n]));
                if (G::KP == 2) {
                    const h8 kl = kt(G::KP - 1);
#pragma unroll
                    for (int n = 0; n < NB; ++n) S[t][n] = mma(kl, hi[s][n], S[t][n]);
                }
            }
        }
    }
}

// v of this wave's columns (and out, the other way): 2 NB lanes a row, 8 columns each
template <class T, int NB>
struct RawV {
    static constexpr int LPR = 2 * NB, ROWS = 64 / LPR, N = C / ROWS;
    typename Vec<T, 8>::raw x[N];
};

// FAST: dk and dv are multiples of 8
template <class T, int NKT, int NB, bool FAST>
__global__ __launch_bounds__(256, 2) void delta_chunk_kernel(const nnsp_delta_args a) {
    using G = Geo<T, NKT, NB>;
    __shared__ Lds<T, NKT, NB> L;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    const int ncb = (a.dv + G::W - 1) / G::W;
    const int cb = blockIdx.x % ncb, h = (blockIdx.x / ncb) % a.value_heads, s = blockIdx.x / ncb / a.value_heads;
    const int hk = h / (a.value_heads / a.key_heads);
    const int n = a.lens ? max(0, min(a.lens[s], a.n_frames)) : a.n_frames;
    const int c0 = cb * G::W + wave * 16 * NB;  // first column of this wave
    const long long so = ((long long)s * a.value_heads + h) * a.dk * a.dv;

    f32x4 S[2 * NKT][NB];
    float sinv[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        sinv[j] = 1.0f;
#pragma unroll
        for (int t = 0; t < 2 * NKT; ++t) S[t][j] = f32x4{0, 0, 0, 0};
    }
    if (a.state_in) {
        const float* p = a.state_in + so;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int t = 0; t < 2 * NKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 32 * (t >> 1) + 8 * g + 4 * (t & 1) + r, col = c0 + 16 * j + l15;
                    const float x = p[min(row, a.dk - 1) * a.dv + min(col, a.dv - 1)];
                    S[t][j][r] = row < a.dk && col < a.dv ? x : 0.0f;
                }
    }

    using RV = RawV<T, NB>;
    const int row = tid >> 2, quarter = tid & 3;
    const int vrow = lane / RV::LPR, vcol = c0 + (lane % RV::LPR) * 8;
    // this thread's places, moved on by a chunk each time
    const T* qp = (const T*)a.q + s * a.q_stride[0] + hk * a.q_stride[2] + row * a.q_stride[1] + quarter * 8;
    const T* kp = (const T*)a.k + s * a.k_stride[0] + hk * a.k_stride[2] + row * a.k_stride[1] + quarter * 8;
    const T* vp = (const T*)a.v + s * a.v_stride[0] + h * a.v_stride[2] + vrow * a.v_stride[1] + vcol;
    T* op = (T*)a.out + s * a.out_stride[0] + h * a.out_stride[2] + vrow * a.out_stride[1] + vcol;
    const float* gp = a.g ? a.g + s * a.g_stride[0] + h * a.g_stride[2] + lane * a.g_stride[1] : nullptr;
    const float* bp = a.beta + s * a.beta_stride[0] + h * a.beta_stride[2] + lane * a.beta_stride[1];
    const long long qs = C * a.q_stride[1], ks = C * a.k_stride[1], vs = RV::ROWS * a.v_stride[1], os = RV::ROWS * a.out_stride[1];
    const long long gs = C * a.g_stride[1], bs = C * a.beta_stride[1];
    const int vleft = a.dv - vcol;

    RawRows<T, NKT> rq, rk;
    RV rv;
    float rg = 0.0f, rb = 0.0f;
    const auto fetch = [&](int t0) {
        const bool live = t0 + row < n;
        fetch_rows<T, NKT, FAST>(rk, kp, quarter, a.dk, live);
        fetch_rows<T, NKT, FAST>(rq, qp, quarter, a.dk, live);
        kp += ks;
        qp += qs;
#pragma unroll
        for (int i = 0; i < RV::N; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) rv.x[i][j] = (T)0.0f;
            const int left = t0 + vrow + RV::ROWS * i < n ? vleft : 0;
            if (FAST) {
                if (left > 0) rv.x[i] = *reinterpret_cast<const typename Vec<T, 8>::type*>(vp);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < left) rv.x[i][j] = vp[j];
            }
            vp += vs;
        }
        if (wave == 0) {
            rg = rb = 0.0f;
            if (t0 + lane < n) {
                if (gp) rg = *gp;
                rb = *bp;
            }
            if (gp) gp += gs;
            bp += bs;
        }
    };
    if (n > 0) fetch(0);
    for (int t0 = 0; t0 < n; t0 += C) {
        const int nt = min(4, (n - t0 + 15) >> 4);
        float ss;
        float inv = stage_rows<T, NKT, G::KP, G::KS>(rk, L.K, row, quarter, ss), len = 1.0f, f = 1.0f;
        f = a.l2norm ? 1.0f / sqrtf(ss + a.eps) : 1.0f;
        len = sqrtf(ss) * f;
        if (quarter == 0) L.kx[row] = inv * f, L.kn[row] = len;
        inv = stage_rows<T, NKT, G::KP, G::KS>(rq, L.Q, row, quarter, ss);
        f = a.scale * (a.l2norm ? 1.0f / sqrtf(ss + a.eps) : 1.0f);
        if (quarter == 0) L.qx[row] = inv * f, L.qn[row] = sqrtf(ss) * fabsf(f);
        if (wave == 0) {
            // running sum of g in 64 bits, in units of log2, kept as two floats: differences of near frames stay exact
            double x = (double)decay_log(rg) * 1.4426950408889634;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double y = __shfl_up(x, d);
                if (lane >= d) x += y;
            }
            L.gh[lane] = (float)x;
            L.gl[lane] = (float)(x - (double)(float)x);
            L.beta[lane] = rb;
        }
        __syncthreads();
        make_tp<T, NKT, NB>(L, wave, here(lane), nt);
#pragma unroll
        for (int i = 0; i < RV::N; ++i)
            *reinterpret_cast<typename Vec<T, 8>::raw*>(&L.V[wave][vrow + RV::ROWS * i][vcol - c0]) = rv.x[i];
        // the wave's own columns: LDS keeps its order within a wave, the compiler has to
        asm volatile("" ::: "memory");
        advance<T, NKT, NB>(L, S, sinv, wave, here(lane), nt, [&] {
            if (t0 + C < n) fetch(t0 + C);
        });
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < RV::N; ++i) {
            const int r = vrow + RV::ROWS * i, left = t0 + r < n ? vleft : 0;
            const auto x = *reinterpret_cast<const typename Vec<T, 8>::raw*>(&L.V[wave][r][vcol - c0]);
            if (FAST) {
                if (left > 0) *reinterpret_cast<typename Vec<T, 8>::type*>(op) = x;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < left) op[j] = x[j];
            }
            op += os;
        }
        __syncthreads();
    }
    if (a.state_out) {
        const int l = here(lane);
        float* p = a.state_out + so;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int t = 0; t < 2 * NKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int rw = 32 * (t >> 1) + 8 * (l >> 4) + 4 * (t & 1) + r, col = c0 + 16 * j + (l & 15);
                    if (rw < a.dk && col < a.dv) p[rw * a.dv + col] = S[t][j][r] * sinv[j];
                }
    }
}

template <class T, int NKT, int NB, bool FAST>
void launch_as(const nnsp_delta_args& a, hipStream_t st) {
    const long long grid = (long long)a.n_streams * a.value_heads * ((a.dv + 64 * NB - 1) / (64 * NB));
    delta_chunk_kernel<T, NKT, NB, FAST><<<dim3((unsigned)grid), dim3(256), 0, st>>>(a);
}
template <class T, int NKT, bool FAST>
void launch_nb(const nnsp_delta_args& a, hipStream_t st) {
    if (a.dv <= 64) launch_as<T, NKT, 1, FAST>(a, st);
    else launch_as<T, NKT, 2, FAST>(a, st);
}
template <class T>
int launch_chunk(const nnsp_delta_args& a, hipStream_t st) {
    if ((a.dk | a.dv) & 7) {
        if (a.dk <= 64) launch_nb<T, 2, false>(a, st);
        else launch_nb<T, 4, false>(a, st);
    } else if (a.dk <= 32) {
        launch_nb<T, 1, true>(a, st);
    } else if (a.dk <= 64) {
        launch_nb<T, 2, true>(a, st);
    } else if (a.dk <= 96) {
        launch_nb<T, 3, true>(a, st);
    } else {
        launch_nb<T, 4, true>(a, st);
    }
    return (int)hipGetLastError();
}

}  // namespace

#endif
