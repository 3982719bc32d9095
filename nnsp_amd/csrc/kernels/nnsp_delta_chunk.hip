// nnsp_delta_chunk.hip -- the gated delta rule over chunks of 64 frames on the
// matrix cores (include/nnsp_seq.h).
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
#include <type_traits>

#include "nnsp_seq_dev.h"
#include "nnsp_seqk.h"

namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr int C = 64;       // frames of a chunk
constexpr int TS = C + 8;   // row of T and P in LDS, halves (16 rows reach all 64 banks)
constexpr int AS = C + 4;   // row of A in LDS, floats

__device__ __forceinline__ f32x4 mma(h8 a, h8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

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

// two accumulator tiles times s as the high and low B operand of a 32-deep product
__device__ __forceinline__ void split(const f32x4& a, const f32x4& b, float s, h8& hi, h8& lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = (i < 4 ? a[i & 3] : b[i & 3]) * s;
        hi[i] = (_Float16)x;
        lo[i] = (_Float16)(x - (float)hi[i]);
    }
}
__device__ __forceinline__ h8 high(const f32x4& a, const f32x4& b, float s) {
    h8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)((i < 4 ? a[i & 3] : b[i & 3]) * s);
    return r;
}

// place of frame j in a row of T and P: the k order of two stacked accumulator tiles
__device__ __forceinline__ int kpos(int j) { return (j & 32) | ((j & 12) << 1) | ((j & 16) >> 2) | (j & 3); }

// 4 rows x 4 columns per lane group, transposed: lane l of 16 gets column l of rows 0 .. 3
__device__ __forceinline__ s4 read_tr(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
}

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
    _Float16 K[G::KP][C][G::KS], Q[G::KP][C][G::KS];
    _Float16 Th[2][C][TS], Ph[G::OP][C][TS];
    union {
        float A[C][AS];            // until T is done
        T V[4][C][G::VS];          // from then on: each wave's columns of v, then of out
    };
    float kx[C], qx[C];            // row factors: norm times 2^-scale
    float gh[C], gl[C], beta[C];   // log2 of the decay up to the frame (two parts), beta
    float fx[C], fk[C], fq[C];     // of K S0, of U into the state, of Q S0
    float ti[C], pi[C];            // 1 / row scales of T and P
    unsigned tmax[C];              // largest |T| of a row
    float D[4][16][20];            // inverses of the diagonal blocks
    float all;                     // decay over the whole chunk
};

// raw rows of q and k on their way to LDS: thread (row, quarter) holds chunks of
// 8 elements quarter, quarter + 4, ...
template <class T, int NKT>
struct RawRows {
    T x[NKT][8];
};
template <class T, int NKT>
__device__ __forceinline__ void fetch_rows(RawRows<T, NKT>& r, const T* p, int quarter, int n, bool live) {
#pragma unroll
    for (int i = 0; i < NKT; ++i) {
        const int c = (quarter + 4 * i) * 8;
        if (live && c + 8 <= n) {
            load_raw(r.x[i], p + c);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) r.x[i][j] = live && c + j < n ? p[c + j] : (T)0.0f;
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
            const float x = (float)r.x[i][j] * s;
            hi[j] = (_Float16)x;
            if (KP == 2) lo[j] = (_Float16)(x - (float)hi[j]);
        }
        const int c = (quarter + 4 * i) * 8;
        *reinterpret_cast<h8*>(&dst[0][row][c]) = hi;
        if (KP == 2) *reinterpret_cast<h8*>(&dst[KP - 1][row][c]) = lo;
    }
    return inv;
}

// tile (mi, mj) of X K^T
template <int NKT, int KP, int KS>
__device__ __forceinline__ f32x4 dot_tile(const _Float16 (*X)[C][KS], const _Float16 (*K)[C][KS], int mi, int mj, int l15, int g) {
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < NKT; ++s) {
        const int c = 32 * s + 8 * g;
        const h8 a = *reinterpret_cast<const h8*>(&X[0][16 * mi + l15][c]), b = *reinterpret_cast<const h8*>(&K[0][16 * mj + l15][c]);
        acc = mma(a, b, acc);
        if (KP == 2) {
            const h8 al = *reinterpret_cast<const h8*>(&X[KP - 1][16 * mi + l15][c]);
            const h8 bl = *reinterpret_cast<const h8*>(&K[KP - 1][16 * mj + l15][c]);
            acc = mma(a, bl, mma(al, b, acc));
        }
    }
    return acc;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// T and P of the staged chunk, by all four waves.  Starts and ends with the
// workgroup together.
template <class T, int NKT, int NB>
__device__ __forceinline__ void make_tp(Lds<T, NKT, NB>& L, int wave, int lane) {
    using G = Geo<T, NKT, NB>;
    const int l15 = lane & 15, g = lane >> 4;
    // rows 16 w .. 16 w + 15 of A; the diagonal's upper half is not read
    for (int j = 0; j <= wave; ++j) {
        const f32x4 acc = dot_tile<NKT, G::KP, G::KS>(L.K, L.K, wave, j, l15, g);
        const int col = 16 * j + l15;
        const float kj = L.kx[col], hj = L.gh[col], lj = L.gl[col];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * wave + 4 * g + r;
            const float d = exp2_fast(fminf((L.gh[row] - hj) + (L.gl[row] - lj), 126.0f));
            L.A[row][col] = L.beta[row] * L.kx[row] * kj * (acc[r] * d);
        }
    }
    __syncthreads();
    if (wave == 0) {
        // the four diagonal blocks, a column of the inverse per lane: x = e - A x from the top
        const int b = 16 * g;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == l15 ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < i; ++j) s = fmaf(-L.A[b + i][b + j], x[j], s);
            x[i] = s;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) L.D[g][i][l15] = x[i];
    } else {
        // P meanwhile: rows of tile 3, 2, and 0 with 1
        for (int mi = wave == 1 ? 3 : wave == 2 ? 2 : 0; mi <= (wave == 1 ? 3 : wave == 2 ? 2 : 1); ++mi) {
            f32x4 p[4];
            float m[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j > mi) continue;
                p[j] = dot_tile<NKT, G::KP, G::KS>(L.Q, L.K, mi, j, l15, g);
                const int col = 16 * j + l15;
                const float kj = L.kx[col], hj = L.gh[col], lj = L.gl[col];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * mi + 4 * g + r;
                    const float d = exp2_fast(fminf((L.gh[row] - hj) + (L.gl[row] - lj), 126.0f));
                    p[j][r] = col <= row ? L.qx[row] * kj * (p[j][r] * d) : 0.0f;
                    m[r] = fmaxf(m[r], fabsf(p[j][r]));
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * mi + 4 * g + r;
                float inv;
                const float s = scale_of(max_row16(m[r]), inv);
                if (l15 == 0) L.pi[row] = inv;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j > (mi | 1)) continue;  // products are 32 frames deep: the tile above the diagonal is read too
                    const float x = j <= mi ? p[j][r] * s : 0.0f;
                    const _Float16 hi = (_Float16)x;
                    L.Ph[0][row][kpos(16 * j + l15)] = hi;
                    if (G::OP == 2) L.Ph[G::OP - 1][row][kpos(16 * j + l15)] = (_Float16)(x - (float)hi);
                }
            }
        }
        if (wave == 3) {
            const int i = lane;
            const float up = exp2_fast(L.gh[i]) ;
            L.fx[i] = L.beta[i] * up * L.kx[i];
            L.fq[i] = up * L.qx[i];
            L.fk[i] = exp2_fast((L.gh[C - 1] - L.gh[i]) + (L.gl[C - 1] - L.gl[i])) * L.kx[i];
            L.tmax[i] = 0;
            if (i == C - 1) L.all = up;
        }
    }
    __syncthreads();
    // block column `wave` of T: T_ij = -T_ii sum over j <= k < i of A_ik T_kj, in 32 bits
    f32x4 t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        t[i] = f32x4{0, 0, 0, 0};
        if (i < wave) continue;
        if (i == wave) {
#pragma unroll
            for (int r = 0; r < 4; ++r) t[i][r] = L.D[i][4 * g + r][l15];
            continue;
        }
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < i; ++k) {
            if (k < wave) continue;
            const f32x4 a = *reinterpret_cast<const f32x4*>(&L.A[16 * i + l15][16 * k + 4 * g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], t[k][r], acc, 0, 0, 0);
        }
        const f32x4 d = *reinterpret_cast<const f32x4*>(&L.D[i][l15][4 * g]);
#pragma unroll
        for (int r = 0; r < 4; ++r) t[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(-d[r], acc[r], t[i], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i >= wave)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float m = max_row16(fabsf(t[i][r]));
                if (l15 == 0) atomicMax(&L.tmax[16 * i + 4 * g + r], __float_as_uint(m));
            }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * i + 4 * g + r;
            if (wave > (i | 1)) continue;
            float inv;
            const float s = scale_of(__uint_as_float(L.tmax[row]), inv);
            const float x = t[i][r] * s;
            const _Float16 hi = (_Float16)x;
            const int c = kpos(16 * wave + l15);
            L.Th[0][row][c] = hi;
            L.Th[1][row][c] = (_Float16)(x - (float)hi);
            if (wave == 0 && l15 == 0) L.ti[row] = inv;
        }
    __syncthreads();
}

// The products with the state for one chunk: this wave's columns.
template <class T, int NKT, int NB>
__device__ __forceinline__ void advance(Lds<T, NKT, NB>& L, f32x4 (&S)[2 * NKT][NB], int wave, int lane) {
    using G = Geo<T, NKT, NB>;
    const int l15 = lane & 15, g = lane >> 4;
    f32x4 R[4][NB], O[4][NB];
    float sinv[NB];
    {
        h8 hi[NKT][NB], lo[NKT][NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float m = 0.0f;
#pragma unroll
            for (int t = 0; t < 2 * NKT; ++t) m = amax4(m, S[t][n]);
            const float s = scale_of(max_xor16_32(m), sinv[n]);
#pragma unroll
            for (int t = 0; t < NKT; ++t) split(S[2 * t][n], S[2 * t + 1][n], s, hi[t][n], lo[t][n]);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            f32x4 x[NB], o[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) x[n] = o[n] = f32x4{0, 0, 0, 0};
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
            const f32x4 b = *reinterpret_cast<const f32x4*>(&L.beta[16 * m + 4 * g]);
            const f32x4 fx = *reinterpret_cast<const f32x4*>(&L.fx[16 * m + 4 * g]);
            const f32x4 fq = *reinterpret_cast<const f32x4*>(&L.fq[16 * m + 4 * g]);
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
                    R[m][n][r] = b[r] * v[r] - fx[r] * (x[n][r] * sinv[n]);
                    O[m][n][r] = fq[r] * (o[n][r] * sinv[n]);
                }
            }
        }
    }
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
            for (int n = 0; n < NB; ++n) u[n] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s <= m / 2; ++s) {
                const h8 th = *reinterpret_cast<const h8*>(&L.Th[0][16 * m + l15][32 * s + 8 * g]);
                const h8 tl = *reinterpret_cast<const h8*>(&L.Th[1][16 * m + l15][32 * s + 8 * g]);
#pragma unroll
                for (int n = 0; n < NB; ++n) u[n] = mma(tl, hi[s][n], mma(th, lo[s][n], mma(th, hi[s][n], u[n])));
            }
            const f32x4 ti = *reinterpret_cast<const f32x4*>(&L.ti[16 * m + 4 * g]);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) U[m][n][r] = u[n][r] * (ti[r] * inv[n]);
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
            f32x4 o[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) o[n] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s <= m / 2; ++s) {
                const h8 ph = *reinterpret_cast<const h8*>(&L.Ph[0][16 * m + l15][32 * s + 8 * g]);
#pragma unroll
                for (int n = 0; n < NB; ++n) o[n] = mma(ph, hi[s][n], o[n]);
                if (G::OP == 2) {
                    const h8 pl = *reinterpret_cast<const h8*>(&L.Ph[G::OP - 1][16 * m + l15][32 * s + 8 * g]);
#pragma unroll
                    for (int n = 0; n < NB; ++n) o[n] = mma(pl, hi[s][n], mma(ph, lo[s][n], o[n]));
                }
            }
            const f32x4 pi = *reinterpret_cast<const f32x4*>(&L.pi[16 * m + 4 * g]);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float o1 = O[m][n][r] + o[n][r] * (pi[r] * inv[n]);
                    L.V[wave][16 * m + 4 * g + r][16 * n + l15] = (T)o1;
                }
        }
    }
    // S1
    {
        h8 hi[2][NB], lo[2][NB];
        float inv[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float m = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const f32x4 fk = *reinterpret_cast<const f32x4*>(&L.fk[16 * t + 4 * g]);
#pragma unroll
                for (int r = 0; r < 4; ++r) U[t][n][r] *= fk[r];
                m = amax4(m, U[t][n]);
            }
            const float s = scale_of(max_xor16_32(m), inv[n]);
#pragma unroll
            for (int t = 0; t < 2; ++t) split(U[2 * t][n], U[2 * t + 1][n], s, hi[t][n], lo[t][n]);
        }
        const float all = L.all;
#pragma unroll
        for (int t = 0; t < 2 * NKT; ++t) {
            f32x4 acc[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) acc[n] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int row = 32 * s + 4 * g + (l15 >> 2), col = 32 * (t >> 1) + 8 * (l15 & 3) + 4 * (t & 1);
                const auto kt = [&](int part) {
                    const s4 a = read_tr(&L.K[part][row][col]), b = read_tr(&L.K[part][row + 16][col]);
                    const h4 x = __builtin_bit_cast(h4, a), y = __builtin_bit_cast(h4, b);
                    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                };
                const h8 k = kt(0);
#pragma unroll
                for (int n = 0; n < NB; ++n) acc[n] = mma(k, lo[s][n], mma(k, hi[s][n], acc[n]));
                if (G::KP == 2) {
                    const h8 kl = kt(G::KP - 1);
#pragma unroll
                    for (int n = 0; n < NB; ++n) acc[n] = mma(kl, hi[s][n], acc[n]);
                }
            }
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[t][n][r] = fmaf(acc[n][r], inv[n], all * S[t][n][r]);
        }
    }
}

// v of this wave's columns (and out, the other way): 2 NB lanes a row, 8
// columns each
template <class T, int NB>
struct RawV {
    static constexpr int LPR = 2 * NB, ROWS = 64 / LPR, N = C / ROWS;
    T x[N][8];
};

template <class T, int NKT, int NB>
__global__ __launch_bounds__(256) void delta_chunk_kernel(const nnsp_delta_args a) {
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
#pragma unroll
    for (int t = 0; t < 2 * NKT; ++t)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 32 * (t >> 1) + 8 * g + 4 * (t & 1) + r, col = c0 + 16 * j + l15;
                S[t][j][r] = a.state_in && row < a.dk && col < a.dv ? a.state_in[so + (long long)row * a.dv + col] : 0.0f;
            }

    const int row = tid >> 2, quarter = tid & 3;
    const T* qp = (const T*)a.q + s * a.q_stride[0] + hk * a.q_stride[2];
    const T* kp = (const T*)a.k + s * a.k_stride[0] + hk * a.k_stride[2];
    const T* vp = (const T*)a.v + s * a.v_stride[0] + h * a.v_stride[2];
    T* op = (T*)a.out + s * a.out_stride[0] + h * a.out_stride[2];
    const float* gp = a.g ? a.g + s * a.g_stride[0] + h * a.g_stride[2] : nullptr;
    const float* bp = a.beta + s * a.beta_stride[0] + h * a.beta_stride[2];

    using RV = RawV<T, NB>;
    const int vrow = lane / RV::LPR, vcol = (lane % RV::LPR) * 8;
    RawRows<T, NKT> rq, rk;
    RV rv;
    float rg = 0.0f, rb = 0.0f;
    const auto fetch = [&](int t0) {
        const long long t = t0 + row;
        fetch_rows<T, NKT>(rk, kp + t * a.k_stride[1], quarter, a.dk, t < n);
        fetch_rows<T, NKT>(rq, qp + t * a.q_stride[1], quarter, a.dk, t < n);
#pragma unroll
        for (int i = 0; i < RV::N; ++i) {
            const long long tv = t0 + vrow + RV::ROWS * i;
            const T* p = vp + tv * a.v_stride[1] + c0 + vcol;
            const int left = tv < n ? a.dv - c0 - vcol : 0;
            if (left >= 8) {
                load_raw(rv.x[i], p);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) rv.x[i][j] = j < left ? p[j] : (T)0.0f;
            }
        }
        if (wave == 0) {
            const long long tg = t0 + lane;
            rg = gp && tg < n ? gp[tg * a.g_stride[1]] : 0.0f;
            rb = tg < n ? bp[tg * a.beta_stride[1]] : 0.0f;
        }
    };
    if (n > 0) fetch(0);
    for (int t0 = 0; t0 < n; t0 += C) {
        float ss;
        float inv = stage_rows<T, NKT, G::KP, G::KS>(rk, L.K, row, quarter, ss);
        if (quarter == 0) L.kx[row] = a.l2norm ? inv / sqrtf(ss + a.eps) : inv;
        inv = stage_rows<T, NKT, G::KP, G::KS>(rq, L.Q, row, quarter, ss);
        if (quarter == 0) L.qx[row] = a.scale * (a.l2norm ? inv / sqrtf(ss + a.eps) : inv);
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
        make_tp<T, NKT, NB>(L, wave, lane);
#pragma unroll
        for (int i = 0; i < RV::N; ++i) {
            T* p = &L.V[wave][vrow + RV::ROWS * i][vcol];
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = rv.x[i][j];
        }
        if (t0 + C < n) fetch(t0 + C);
        // the wave's own columns: LDS keeps its order within a wave, the compiler has to
        asm volatile("" ::: "memory");
        advance<T, NKT, NB>(L, S, wave, lane);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < RV::N; ++i) {
            const int r = vrow + RV::ROWS * i, left = t0 + r < n ? a.dv - c0 - vcol : 0;
            T* p = op + (long long)(t0 + r) * a.out_stride[1] + c0 + vcol;
            T x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = L.V[wave][r][vcol + j];
            if (left >= 8) {
                typename Vec<T, 8>::raw v;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = x[j];
                *reinterpret_cast<typename Vec<T, 8>::type*>(p) = v;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < left) p[j] = x[j];
            }
        }
        __syncthreads();
    }
    if (a.state_out) {
#pragma unroll
        for (int t = 0; t < 2 * NKT; ++t)
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int rw = 32 * (t >> 1) + 8 * g + 4 * (t & 1) + r, col = c0 + 16 * j + l15;
                    if (rw < a.dk && col < a.dv) a.state_out[so + (long long)rw * a.dv + col] = S[t][j][r];
                }
    }
}

template <class T, int NKT, int NB>
void launch_as(const nnsp_delta_args& a, hipStream_t st) {
    const long long grid = (long long)a.n_streams * a.value_heads * ((a.dv + 64 * NB - 1) / (64 * NB));
    delta_chunk_kernel<T, NKT, NB><<<dim3((unsigned)grid), dim3(256), 0, st>>>(a);
}
template <class T, int NKT>
void launch_nb(const nnsp_delta_args& a, hipStream_t st) {
    if (a.dv <= 64) launch_as<T, NKT, 1>(a, st);
    else launch_as<T, NKT, 2>(a, st);
}
template <class T>
void launch_nkt(const nnsp_delta_args& a, hipStream_t st) {
    if (a.dk <= 32) launch_nb<T, 1>(a, st);
    else if (a.dk <= 64) launch_nb<T, 2>(a, st);
    else if (a.dk <= 96) launch_nb<T, 3>(a, st);
    else launch_nb<T, 4>(a, st);
}

}  // namespace

extern "C" int nnspk_launch_delta_chunk(const nnsp_delta_args* a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    if (a->dtype == NNSP_BF16) launch_nkt<__bf16>(*a, st);
    else if (a->dtype == NNSP_F16) launch_nkt<_Float16>(*a, st);
    else launch_nkt<float>(*a, st);
    return (int)hipGetLastError();
}
