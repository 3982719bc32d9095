// nnsp_delta_chunk.h -- the gated delta rule over chunks of frames on the
// matrix cores (include/nnsp_seq.h); one .hip file per element type launches it.
//
// Within a chunk, with G_i the sum of g up to frame i and S0 the state before it,
//
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j   (j < i)        T = (I + A)^-1
//   U    = T (beta V - beta e^G (K S0))
//   O    = scale (e^G (Q S0) + P U)         P_ij = e^(G_i - G_j) q_i . k_j (j <= i)
//   S1   = e^(G_n) S0 + K^T (e^(G_n - G) U)       (n the chunk's last frame)
//
// which is the rule of a chunk's frames with the recurrence left in one
// triangular inverse.  T and P need no state; the rest is five matrix products.
//
// Numbers.  The state, T and U are 32-bit values, and the matrix cores take 16
// bits: each is scaled by a power of two and split into an fp16 high and low
// part, 22 bits in all, and products keep hi hi + hi lo + lo hi, accumulated in
// 32 bits.  A column has powers of its own, as it is a recurrence of its own:
// neither its precision nor its range depends on the columns beside it, and what
// is not finite stays in it.  They come from the column's largest magnitude or
// from a bound.  An fp16 pair is good to 2^-23 of its value, or to 2^-25, which is
// 2^-39 of what is scaled to 2^14; a bound is at most 64 times the largest term of
// the sum it is of (and 2^5 more where R's own was a bound), so that this stays
// below 2^-28 of that term, and adding the sum up in 32 bits loses 2^-24 of it.
// T has a power a row tile, shared by all columns.  q and k go in with their rows
// scaled too: fp16 and bf16 in one part (exact down to 2^-19 and 2^-28 of a row's
// largest, to 2^-30 and 2^-39 of it below), fp32 in two.  All other factors
// (norms, decays, beta) multiply in 32 bits outside the products.
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

// frames of a chunk: 64 where a chain of chunks is what takes time, 32 where
// many streams fill the device and registers and LDS decide how well (100 frames
// of 8192 streams, 2 heads of 64 x 64: chunks of 64 667 us, of 32 607 us then)
constexpr int C = 64, CF = 32;
// images of a slab, inside the 256 MB cache behind the L2s (16384 frames of 32
// heads of 128 x 128, us: 32 MB 737, 96 MB 607, 200 MB 625; fp32 1295, 1250, 1290)
constexpr long long DELTA_SLAB_BYTES = 96ll << 20;

// sizes of a call in two passes
struct DeltaSplit {
    int chunks, slab;                           // chunks of the call, of a slab
    long long kq_bytes, tp_bytes, state_bytes;  // images of a chunk; the state between slabs
    long long bytes() const { return state_bytes + slab * (kq_bytes + tp_bytes); }
};

__device__ __forceinline__ f32x4 mma(h8 a, h8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// power of two that takes m's magnitude to [2^14, 2^15), and its inverse
__device__ __forceinline__ float scale_of(float m, float& inv) {
    const int e = (__float_as_int(m) >> 23) & 255;
    const int s = min(max(268 - e, 1), 253);
    inv = __int_as_float((254 - s) << 23);
    return __int_as_float(s << 23);
}
// 1 / x of a power of two from 2^-126 to 2^126
__device__ __forceinline__ float inverse2(float x) { return __int_as_float((254 << 23) - __float_as_int(x)); }
// 0, or NaN of an infinite magnitude: a scale that holds an infinity would leave
// the values beside it 0, so it is made to show
__device__ __forceinline__ float poison(float m) { return m * 0.0f; }
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
// largest over the wave
__device__ __forceinline__ float wave_max(float x) {
    return max_xor16_32(max_dpp<0x128>(max_dpp<0x141>(max_dpp<0x4e>(max_dpp<0xb1>(x)))));
}
__device__ __forceinline__ float amax4(float m, const f32x4& x) {
    return fmaxf(fmaxf(fmaxf(m, fabsf(x[0])), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
}

// the value of the lane N before in the row of 16; the first N keep `first`
template <int N>
__device__ __forceinline__ float row_shr(float x, float first) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(first), __float_as_int(x), 0x110 + N, 0xf, 0xf, false));
}
template <int N>
__device__ __forceinline__ double row_shr(double x) {
    const long long b = __builtin_bit_cast(long long, x);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)b, 0x110 + N, 0xf, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), 0x110 + N, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (unsigned)lo | (long long)hi << 32);
}
__device__ __forceinline__ double lane_of(double x, int l) {
    const long long b = __builtin_bit_cast(long long, x);
    const int lo = __builtin_amdgcn_readlane((int)b, l), hi = __builtin_amdgcn_readlane((int)(b >> 32), l);
    return __builtin_bit_cast(double, (unsigned)lo | (long long)hi << 32);
}
// sum and minimum over the lanes up to this one of each group of C (32, 64)
template <int C>
__device__ __forceinline__ double scan_sum(double x, int lane) {
    x += row_shr<1>(x);
    x += row_shr<2>(x);
    x += row_shr<4>(x);
    x += row_shr<8>(x);
    const double a = lane_of(x, 15), b = lane_of(x, 47);
    if (C == 32) return lane & 16 ? x + (lane & 32 ? b : a) : x;
    const double m = lane_of(x, 31) + a;
    return x + (lane < 16 ? 0.0 : lane < 32 ? a : lane < 48 ? m : m + b);
}
template <int C>
__device__ __forceinline__ float scan_min(float x, int lane) {
    x = fminf(x, row_shr<1>(x, x));
    x = fminf(x, row_shr<2>(x, x));
    x = fminf(x, row_shr<4>(x, x));
    x = fminf(x, row_shr<8>(x, x));
    const auto of = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); };
    const float a = of(15), b = of(47);
    if (C == 32) return lane & 16 ? fminf(x, lane & 32 ? b : a) : x;
    const float m = fminf(of(31), a);
    return lane < 16 ? x : fminf(x, lane < 32 ? a : lane < 48 ? m : fminf(m, b));
}

// Everything this wave has asked of global memory is there.  Put before a loop
// and before its stores, whose completion would otherwise be waited for together
// with the loads that came before them (two passes over 16384 frames of 32 heads
// of 128 x 128: 641 -> 616 us).
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// a copy the compiler knows nothing about: LDS addresses made of it are not
// kept in registers from chunk to chunk
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// x s rounded to fp16, as one mixed-precision fma with a zero that the compiler cannot see through
__device__ __forceinline__ _Float16 half_of(float x, float s) {
    float zero = 0.0f;
    asm("" : "+s"(zero));
    return (_Float16)fmaf(x, s, zero);
}
// two accumulator tiles times their rows' factors s as the high and low B
// operand of a 32-deep product
__device__ __forceinline__ void split(const f32x4& a, const f32x4& b, const f32x4& sa, const f32x4& sb, h8& hi, h8& lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) hi[i] = half_of(i < 4 ? a[i & 3] : b[i & 3], i < 4 ? sa[i & 3] : sb[i & 3]);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        lo[i] = (_Float16)fmaf(i < 4 ? a[i & 3] : b[i & 3], i < 4 ? sa[i & 3] : sb[i & 3], -(float)hi[i]);
}
__device__ __forceinline__ f32x4 all4(float x) { return f32x4{x, x, x, x}; }

// 4 rows x 4 columns per lane group, transposed: lane l of 16 gets column l of rows 0 .. 3
__device__ __forceinline__ s4 read_tr(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
}

// T and P in LDS, in the k order of two stacked accumulator tiles: row tiles 0
// and 1 hold 32 frames a row, 2 and 3 (of 64-frame chunks) all 64; 8 halves of
// padding spread 16 rows over all banks
template <int C>
struct Tri {
    alignas(16) _Float16 x[32 * 40 + (C - 32) * 72];
    static __device__ __forceinline__ int row(int m, int l15) {
        return m < 2 ? (16 * m + l15) * 40 : 1280 + (16 * m - 32 + l15) * 72;
    }
    // frames 32 s + 8-element group g of row 16 m + l15
    __device__ __forceinline__ h8 operand(int m, int l15, int s, int g) const {
        return *reinterpret_cast<const h8*>(x + row(m, l15) + 32 * s + 8 * g);
    }
    // frames 16 j + 4 g .. + 3 of row 16 m + l15
    __device__ __forceinline__ void put(int m, int l15, int j, int g, h4 v) {
        *reinterpret_cast<h4*>(x + row(m, l15) + 32 * (j >> 1) + 8 * g + 4 * (j & 1)) = v;
    }
};

template <class T, int NKT, int NB>
struct Geo {
    static constexpr bool WIDE = std::is_same<T, float>::value;       // 32-bit input
    static constexpr int KP = WIDE ? 2 : 1;                           // parts of q and k
    static constexpr int VS = 16 * NB + 4;                            // row of a wave's V, elements
};

// q and k of a chunk as the products take them
template <class T, int NKT, int C>
struct KQ {
    static constexpr int KP = std::is_same<T, float>::value ? 2 : 1, KS = NKT * 32 + 8;
    // 64 elements of K at most: rows are scaled to a length below 2^6 in fp16, to a largest element below 2^15 else
    static constexpr float BOUND64 = std::is_same<T, _Float16>::value ? 0x1p12f : 0x1p21f;
    alignas(16) _Float16 K[KP][C][KS], Q[KP][C][KS];
};
// what else a chunk's products take; e() is a decay, G the sum of g
template <class T, int C>
struct TP {
    Tri<C> P_[2];
    alignas(16) float beta[C], fx[C], fk[C], fq[C];  // factors of v, K S0, U into the state, Q S0
    alignas(16) float pi[C];                         // 2^-scale of P's rows
    float ti[4];                                     // 2^-scale of T's row tiles
    float all, fkmax;                                // decay over the whole chunk; largest fk
    float bmax, xmax;                                // largest |beta|; |beta e(G) k^ . x| is at most xmax |x|_max
    Tri<C> T_[2];                                    // last: what T is made from lies here and beyond until then
};
// what making T and P takes besides; s and e are the first and last frame of a frame's 16
template <int C>
struct Make {
    alignas(16) float kx[C], qx[C], kn[C], qn[C];  // norm times 2^-scale, length after the norm
    alignas(16) float gh[C], gl[C];                // log2 of the decay up to the frame (two parts)
    alignas(16) float ab[C], ar[C];                // A rows: beta kx, times e(G - G_s)
    alignas(16) float pb[C], pr[C];                // P rows: qx 2^scale, times e(G - G_s)
    alignas(16) float kc[C];                       // columns of both: kx e(G_e - G)
};
template <int C>
struct TriA {
    alignas(16) float A[C][C + 4];  // A transposed
};
template <int C>
struct Diag {
    alignas(16) float D[C / 16][16][20];  // transposed inverses of the diagonal blocks
};
static_assert(sizeof(Diag<32>) <= 2 * sizeof(Tri<32>), "the inverses lie where T is written afterwards");

// raw rows of q and k on their way to LDS, PR threads a row: thread (row, part)
// holds chunks of 8 elements part, part + PR, ...
template <class T, int NKT, int PR>
struct RawRows {
    static constexpr int N = (4 * NKT + PR - 1) / PR;
    typename Vec<T, 8>::raw x[N];
};
template <bool FAST, class T, int NKT, int PR>
__device__ __forceinline__ void fetch_rows(RawRows<T, NKT, PR>& r, const T* p, int part, int n, bool live) {
#pragma unroll
    for (int i = 0; i < r.N; ++i) {
        const int c = (part + PR * i) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) r.x[i][j] = (T)0.0f;
        if (FAST) {
            if (live && c < n) r.x[i] = *reinterpret_cast<const typename Vec<T, 8>::type*>(p + 8 * PR * i);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (live && c + j < n) r.x[i][j] = p[8 * PR * i + j];
        }
    }
}
// scaled fp16 parts to LDS; returns 2^-scale (0 of a row of zeros) and the sum of
// the scaled values' squares, which stays in range however loud or faint the row is
template <int KP, int C, int KS, class T, int NKT, int PR>
__device__ __forceinline__ float stage_rows(const RawRows<T, NKT, PR>& r, _Float16 (*dst)[C][KS], int row, int part, float& ss) {
    constexpr int N = RawRows<T, NKT, PR>::N;
    const auto sum = [](float x) {
        x = add_xor2(add_xor1(x));
        if (PR >= 8) x = add_mirror4(x);
        return PR >= 16 ? add_xor8(x) : x;
    };
    ss = 0.0f;
    float inv;
    if constexpr (std::is_same<T, _Float16>::value) {
        // rows to a length of 2^5 .. 2^6, by the exponent of the sum of squares (which fp16 keeps in fp32's range)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const h2 x = {r.x[i][j], r.x[i][j + 1]};
                ss = __builtin_amdgcn_fdot2(x, x, ss, false);
            }
        ss = sum(ss);
        const int e = min(max(5 - (((__float_as_int(ss) >> 23) - 127) >> 1), -14), 15);
        const _Float16 s = __builtin_bit_cast(_Float16, (unsigned short)((15 + e) << 10));
        inv = ss > 0.0f ? __int_as_float((127 - e) << 23) : 0.0f;
        ss *= __int_as_float((127 + 2 * e) << 23);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (4 * NKT % PR == 0 || part + PR * i < 4 * NKT) *reinterpret_cast<h8*>(&dst[0][row][(part + PR * i) * 8]) = r.x[i] * s;
    } else {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf((float)r.x[i][j]));
        m = max_dpp<0x4e>(max_dpp<0xb1>(m));
        if (PR >= 8) m = max_dpp<0x141>(m);
        if (PR >= 16) m = max_dpp<0x128>(m);
        const float s = scale_of(m, inv);
        if (m == 0.0f) inv = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            h8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = (float)r.x[i][j] * s;
                ss = fmaf(x, x, ss);
                hi[j] = (_Float16)x;
                if (KP == 2) lo[j] = (_Float16)(x - (float)hi[j]);
            }
            const int c = (part + PR * i) * 8;
            if (4 * NKT % PR != 0 && c >= 32 * NKT) continue;
            *reinterpret_cast<h8*>(&dst[0][row][c]) = hi;
            if (KP == 2) *reinterpret_cast<h8*>(&dst[KP - 1][row][c]) = lo;
        }
        ss = sum(ss);
    }
    return inv;
}

// tile (mi, mj) of X Y^T
template <int NKT, int KP, int C, int KS>
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

// Factors of the staged frames, a frame a lane (of a chunk of 32 twice): part 0
// those of A, part 1 those of P, part 2 those of the products with the state.
//
// A decay between two frames of different 16s is a product of three that are
// each at most 1 (to the end of the column's 16, between, from the start of
// the row's), so it costs two multiplications an element; within a 16 it is an
// exponential of the difference.  P's row scale comes from a bound (lengths of
// q and k, the largest decay ratio), which an fp16's exponent has room for.
template <int NKT, class T, int C>
__device__ __forceinline__ void make_factors(const KQ<T, NKT, C>&, TP<T, C>& Y, Make<C>& M, int part, int lane) {
    const int i = lane & (C - 1), s = i & ~15, e = i | 15;
    const float h = M.gh[i], l = M.gl[i], kx = M.kx[i];
    if (part == 0) {
        const float b = Y.beta[i] * kx, r = exp2_fast((h - M.gh[s]) + (l - M.gl[s]));
        M.ab[i] = b;
        M.ar[i] = b * r;
        M.kc[i] = exp2_fast((M.gh[e] - h) + (M.gl[e] - l)) * kx;
    } else if (part == 1) {
        // largest decay ratio of a row: e(G_i - min over j <= i of G_j); largest length of a key
        const float lo = scan_min<C>(h, lane), kn = wave_max(M.kn[i]);
        float inv;
        const float qx = M.qx[i], sc = scale_of(M.qn[i] * kn * exp2_fast(fminf(h - lo, 120.0f)), inv);
        Y.pi[i] = inv + poison(kn);
        M.pb[i] = qx * sc;
        M.pr[i] = qx * sc * exp2_fast((h - M.gh[s]) + (l - M.gl[s]));
    } else {
        const float up = exp2_fast(h), b = Y.beta[i];
        Y.fx[i] = b * up * kx;
        Y.fq[i] = up * M.qx[i];
        const float fk = exp2_fast((M.gh[C - 1] - h) + (M.gl[C - 1] - l)) * kx;
        Y.fk[i] = fk;
        const float m = wave_max(fk);
        if (i == C - 1) Y.all = up, Y.fkmax = m;
        if (C == 64) {  // bounds for a scan
            const float bm = wave_max(fabsf(b)), x = wave_max(fabsf(b) * up * M.kn[i]) * sqrtf(32.0f * NKT);
            if (i == C - 1) Y.bmax = bm, Y.xmax = x;
        }
    }
}

// tile (mi, j) of A from that of K K^T
template <int C>
__device__ __forceinline__ void put_a(const Make<C>& M, TriA<C>& A, const f32x4& acc, int mi, int j, int l15, int g) {
    const int col = 16 * j + l15, row = 16 * mi + 4 * g;
    f32x4 f;
    if (j == mi) {
        const f32x4 h = ld4(&M.gh[row]), l = ld4(&M.gl[row]), b = ld4(&M.ab[row]);
        const float hj = M.gh[col], lj = M.gl[col], kj = M.kx[col];
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = exp2_fast(fminf((h[r] - hj) + (l[r] - lj), 120.0f)) * (b[r] * kj);
    } else {
        const int a = 16 * mi, e = 16 * j + 15;
        f = ld4(&M.ar[row]) * (M.kc[col] * exp2_fast((M.gh[a] - M.gh[e]) + (M.gl[a] - M.gl[e])));
    }
    *reinterpret_cast<f32x4*>(&A.A[col][row]) = acc * f;
}

// tile (mi, j) of P from that of K Q^T (so that a lane has 4 frames of a row); zeros above the diagonal
template <class T, int C>
__device__ __forceinline__ void put_p(TP<T, C>& Y, const Make<C>& M, const f32x4& p, int mi, int j, int l15, int g) {
    h4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    if (j <= mi) {
        const int row = 16 * mi + l15, col = 16 * j + 4 * g;
        f32x4 f;
        if (j == mi) {
            const f32x4 h = ld4(&M.gh[col]), l = ld4(&M.gl[col]), k = ld4(&M.kx[col]);
            const float pb = M.pb[row], hi = M.gh[row], li = M.gl[row];
#pragma unroll
            for (int r = 0; r < 4; ++r) f[r] = exp2_fast(fminf((hi - h[r]) + (li - l[r]), 120.0f)) * (k[r] * pb);
        } else {
            const int s = 16 * mi, e = 16 * j + 15;
            f = ld4(&M.kc[col]) * (M.pr[row] * exp2_fast((M.gh[s] - M.gh[e]) + (M.gl[s] - M.gl[e])));
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float x = j == mi && col + r > row ? 0.0f : p[r] * f[r];
            a[r] = (_Float16)x;
            b[r] = (_Float16)fmaf(p[r], f[r], -(float)a[r]);
            if (j == mi && col + r > row) b[r] = (_Float16)0.0f;
        }
    }
    Y.P_[0].put(mi, l15, j, g, a);
    Y.P_[1].put(mi, l15, j, g, b);
}

// block (mi, j) of T, transposed, times s
template <class T, int C>
__device__ __forceinline__ void put_t(TP<T, C>& Y, const f32x4& t, float s, int mi, int j, int l15, int g) {
    h4 a, b;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        a[r] = (_Float16)(t[r] * s);
        b[r] = (_Float16)fmaf(t[r], s, -(float)a[r]);
    }
    Y.T_[0].put(mi, l15, j, g, a);
    Y.T_[1].put(mi, l15, j, g, b);
}

// the inverses of the diagonal blocks by one wave, a column per lane, by substitution from the top
template <int C>
__device__ __forceinline__ void invert_diagonal(const TriA<C>& A, Diag<C>& D, int g, int l15) {
    const int k = g & (C / 16 - 1), b = 16 * k;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = i == l15 ? 1.0f : 0.0f;
    // column j of A, what is below the diagonal, two steps ahead of its use (all at once would be 144 registers)
    f32x4 a[3][4];
    const auto column = [&](int j) {
#pragma unroll
        for (int q = (j + 1) / 4; q < 4; ++q) a[j % 3][q] = ld4(&A.A[b + j][b + 4 * q]);
    };
    column(0);
    column(1);
#pragma unroll
    for (int j = 0; j < 15; ++j) {
        if (j + 2 < 15) column(j + 2);
        asm volatile("" : "+v"(x[j]) : : "memory");
#pragma unroll
        for (int i = j + 1; i < 16; ++i) x[i] = fmaf(-a[j % 3][i / 4][i % 4], x[j], x[i]);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<f32x4*>(&D.D[k][l15][4 * q]) = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
}

// Everything of a staged chunk of 64 that needs no state, by four waves.  Starts
// and ends with the workgroup together.  A may lie where T is written.
template <class T, int NKT>
__device__ __forceinline__ void make_tp(const KQ<T, NKT, 64>& X, TP<T, 64>& Y, Make<64>& M, Diag<64>& D, TriA<64>& A, int wave,
                                        int lane) {
    constexpr int KP = KQ<T, NKT, 64>::KP;
    const int l15 = lane & 15, g = lane >> 4;
    f32x4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j <= wave) acc[j] = dot_tile<NKT, KP>(X.K, X.K, wave, j, l15, g);
    if (wave < 3) make_factors<NKT>(X, Y, M, wave, lane);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j > wave) continue;
        put_a(M, A, acc[j], wave, j, l15, g);
    }
    __syncthreads();
    if (wave == 0) {
        invert_diagonal(A, D, g, l15);
    } else {
        // P meanwhile: rows of tile 3, 2, and 1 with 0
        const int first = wave == 1 ? 3 : wave == 2 ? 2 : 0, last = wave == 3 ? 1 : first;
        for (int mi = first; mi <= last; ++mi)
            for (int j = 0; j <= (mi | 1); ++j)
                put_p(Y, M, j <= mi ? dot_tile<NKT, KP>(X.K, X.Q, j, mi, l15, g) : f32x4{0, 0, 0, 0}, mi, j, l15, g);
    }
    __syncthreads();
    // block row i = wave of T, transposed: N_ij = -T_jj^T sum over j < k <= i of A_kj^T N_ik, in 32 bits
    f32x4 t[4];
    float m = 0.0f;
#pragma unroll
    for (int j = 3; j >= 0; --j) {
        t[j] = f32x4{0, 0, 0, 0};
        if (j > wave) continue;
        if (j == wave) {
#pragma unroll
            for (int r = 0; r < 4; ++r) t[j][r] = D.D[j][4 * g + r][l15];
        } else {
            f32x4 y = {0, 0, 0, 0};
#pragma unroll
            for (int k = j + 1; k < 4; ++k) {
                if (k > wave) continue;
                const f32x4 a = ld4(&A.A[16 * j + l15][16 * k + 4 * g]);
#pragma unroll
                for (int r = 0; r < 4; ++r) y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], t[k][r], y, 0, 0, 0);
            }
            const f32x4 d = ld4(&D.D[j][l15][4 * g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) t[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(-d[r], y[r], t[j], 0, 0, 0);
        }
        m = amax4(m, t[j]);
    }
    __syncthreads();
    {
        float inv;
        m = wave_max(m);
        const float s = scale_of(m, inv);
        if (lane == 0) Y.ti[wave] = inv + poison(m);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j <= (wave | 1)) put_t(Y, t[j], s, wave, j, l15, g);
    }
    __syncthreads();
}

// T of a chunk of 32 by one wave: both diagonal inverses, then N_10 = -T_00^T A_10^T T_11^T
template <class T, class F>
__device__ __forceinline__ void make_t(TP<T, 32>& Y, const TriA<32>& A, int lane, const F& mid) {
    const int l15 = lane & 15, g = lane >> 4;
    Diag<32>& D = *reinterpret_cast<Diag<32>*>(Y.T_);
    invert_diagonal(A, D, g, l15);
    mid();
    asm volatile("" ::: "memory");  // LDS keeps its order within a wave, the compiler has to
    f32x4 t0, t1, y = {0, 0, 0, 0}, t = {0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < 4; ++r) t0[r] = D.D[0][4 * g + r][l15], t1[r] = D.D[1][4 * g + r][l15];
    const f32x4 a = ld4(&A.A[l15][16 + 4 * g]), d = ld4(&D.D[0][l15][4 * g]);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int r = 0; r < 4; ++r) y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], t1[r], y, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) t = __builtin_amdgcn_mfma_f32_16x16x4f32(-d[r], y[r], t, 0, 0, 0);
    float inv;
    const float m = wave_max(amax4(amax4(amax4(0.0f, t0), t1), t)), s = scale_of(m, inv);
    if (lane == 0) Y.ti[0] = inv + poison(m);
    put_t(Y, t0, s, 0, 0, l15, g);
    put_t(Y, f32x4{0, 0, 0, 0}, s, 0, 1, l15, g);
    put_t(Y, t, s, 1, 0, l15, g);
    put_t(Y, t1, s, 1, 1, l15, g);
}

// accumulator tile n of 16 staged rows of v
template <class T, int VS>
__device__ __forceinline__ f32x4 tile_of(const T (*V)[VS], int n, int l15, int g) {
    f32x4 v;
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = V[4 * g + r][16 * n + l15];
    } else {
        const auto t = __builtin_bit_cast(typename Vec<T, 4>::raw, read_tr(&V[4 * g + (l15 >> 2)][16 * n + 4 * (l15 & 3)]));
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = (float)t[r];
    }
    return v;
}

// K S0, R and Q S0 of a chunk of 32 with nt live tiles of 16 frames, for this
// wave's columns.  S holds the state times 1 / sinv, powers of two; a lane's
// scales are those of its column.
template <class T, int NKT, int NB>
struct Chunk {
    using G = Geo<T, NKT, NB>;
    f32x4 R[2][NB], O[2][NB];
    float smax[NB], rmax[NB];

    __device__ __forceinline__ void first(const KQ<T, NKT, 32>& X, const TP<T, 32>& Y, T (*V)[G::VS], const f32x4 (&S)[2 * NKT][NB],
                                          const float (&sinv)[NB], int lane, int nt) {
        const int l15 = lane & 15, g = lane >> 4;
        const f32x4 zero = {0, 0, 0, 0};
        h8 hi[NKT][NB], lo[NKT][NB];
        float sout[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float m = 0.0f, inv;
#pragma unroll
            for (int t = 0; t < 2 * NKT; ++t) m = amax4(m, S[t][n]);
            smax[n] = max_xor16_32(m);
            rmax[n] = 0.0f;
            const float sc = scale_of(smax[n], inv);
            sout[n] = fmaf(inv, sinv[n], poison(smax[n]));
#pragma unroll
            for (int t = 0; t < NKT; ++t) split(S[2 * t][n], S[2 * t + 1][n], all4(sc), all4(sc), hi[t][n], lo[t][n]);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (m >= nt) {
#pragma unroll
                for (int n = 0; n < NB; ++n) R[m][n] = zero;
                continue;
            }
            f32x4 x[NB], o[NB];
#pragma unroll
            for (int s = 0; s < NKT; ++s) {
                const int c = 32 * s + 8 * g;
                const h8 k = *reinterpret_cast<const h8*>(&X.K[0][16 * m + l15][c]);
                const h8 q = *reinterpret_cast<const h8*>(&X.Q[0][16 * m + l15][c]);
                h8 kl, ql;
                if (G::KP == 2) {
                    kl = *reinterpret_cast<const h8*>(&X.K[G::KP - 1][16 * m + l15][c]);
                    ql = *reinterpret_cast<const h8*>(&X.Q[G::KP - 1][16 * m + l15][c]);
                }
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    x[n] = mma(k, lo[s][n], mma(k, hi[s][n], s ? x[n] : zero));
                    o[n] = mma(q, lo[s][n], mma(q, hi[s][n], s ? o[n] : zero));
                    if (G::KP == 2) {
                        x[n] = mma(kl, hi[s][n], x[n]);
                        o[n] = mma(ql, hi[s][n], o[n]);
                    }
                }
            }
            const f32x4 b = ld4(&Y.beta[16 * m + 4 * g]), f = ld4(&Y.fx[16 * m + 4 * g]);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const f32x4 v = tile_of<T>(V + 16 * m, n, l15, g) * b, fx = f * -sout[n];
#pragma unroll
                for (int r = 0; r < 4; ++r) R[m][n][r] = fmaf(fx[r], x[n][r], v[r]);
                O[m][n] = o[n] * (ld4(&Y.fq[16 * m + 4 * g]) * sout[n]);
                rmax[n] = amax4(rmax[n], R[m][n]);
            }
        }
    }

    // U, the output (into V) and the state after the chunk; mid() is called once on the way
    template <class F>
    __device__ __forceinline__ void second(const KQ<T, NKT, 32>& X, const TP<T, 32>& Y, T (*V)[G::VS], f32x4 (&S)[2 * NKT][NB],
                                           float (&sinv)[NB], int lane, int nt, const F& mid) {
        const int l15 = lane & 15, g = lane >> 4;
        const f32x4 zero = {0, 0, 0, 0};
        f32x4 u[2][NB];  // U = u ti rinv, where |u| is at most 32 products of 2^30
        float rs[NB], ti[NB];
        h8 hi[NB], lo[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float inv;
            rmax[n] = max_xor16_32(rmax[n]);
            rs[n] = scale_of(rmax[n], inv);
            ti[n] = fmaf(Y.ti[0], inv, poison(rmax[n]));
            split(R[0][n], R[1][n], all4(rs[n]), all4(rs[n]), hi[n], lo[n]);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const h8 th = Y.T_[0].operand(m, l15, 0, g), tl = Y.T_[1].operand(m, l15, 0, g);
#pragma unroll
            for (int n = 0; n < NB; ++n) u[m][n] = mma(tl, hi[n], mma(th, lo[n], mma(th, hi[n], zero)));
        }
#pragma unroll
        // u to below 2^14: times 2^-22
        for (int n = 0; n < NB; ++n) split(u[0][n], u[1][n], all4(0x1p-22f), all4(0x1p-22f), hi[n], lo[n]);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (m >= nt) continue;
            const h8 ph = Y.P_[0].operand(m, l15, 0, g), pl = Y.P_[1].operand(m, l15, 0, g);
            f32x4 o[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                o[n] = mma(ph, hi[n], zero);
                o[n] = mma(pl, hi[n], mma(ph, lo[n], o[n]));
            }
            const f32x4 p = ld4(&Y.pi[16 * m + 4 * g]);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const f32x4 pi = p * (ti[n] * 0x1p22f);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    V[16 * m + 4 * g + r][16 * n + l15] = (T)fmaf(o[n][r], pi[r], O[m][n][r]);
            }
        }
        mid();
        // S1, accumulated onto the decayed state in the scale s of U fk; where U is next to nothing, in 2^13 of the
        // decayed state's own, so that neither leaves its range (2^100 at most: the state's factor stays finite)
        const float all = Y.all;
        float zi;
        const float z = scale_of(Y.fkmax, zi) * 0x1p-36f * inverse2(Y.ti[0]);
        const f32x4 fk0 = ld4(&Y.fk[4 * g]), fk1 = ld4(&Y.fk[16 + 4 * g]);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float li;
            const float low = scale_of(fmaxf(smax[n] * sinv[n] * (all * 0x1p-13f), 0x1p-86f), li);
            const float s = fminf(z * rs[n], low), d = all * s * sinv[n];  // true U fk times s = u fk (ti s)
            sinv[n] = inverse2(s);
            const f32x4 f0 = fk0 * (ti[n] * s), f1 = fk1 * (ti[n] * s);
            split(u[0][n], u[1][n], f0, f1, hi[n], lo[n]);
#pragma unroll
            for (int t = 0; t < 2 * NKT; ++t) S[t][n] *= d;
        }
#pragma unroll
        for (int t = 0; t < 2 * NKT; ++t) {
            const int row = 4 * g + (l15 >> 2), col = 32 * (t >> 1) + 8 * (l15 & 3) + 4 * (t & 1);
#pragma unroll
            for (int part = 0; part < G::KP; ++part) {
                const h4 x = __builtin_bit_cast(h4, read_tr(&X.K[part][row][col]));
                const h4 y = __builtin_bit_cast(h4, read_tr(&X.K[part][row + 16][col]));
                const h8 k = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    S[t][n] = mma(k, hi[n], S[t][n]);
                    if (part == 0) S[t][n] = mma(k, lo[n], S[t][n]);
                }
            }
        }
    }
};

// Where element r of accumulator tile t, j lies in the head's state: base + at,
// base the same for all lanes, `at` kept inside the state, `in` if it is one of it.
// live: the tile has any.  FAST: dk and dv are multiples of 8.
struct Spot {
    int base;
    unsigned at;
    bool in, live;
};
template <bool FAST>
__device__ __forceinline__ Spot spot(const nnsp_delta_args& a, int c0, int t, int j, int r, int lane) {
    const int l15 = lane & 15, g = lane >> 4, r0 = 32 * (t >> 1), row = r0 + 4 * (t & 1) + r, col = c0 + 16 * j;
    if (FAST)
        return {row * a.dv + col, (unsigned)(min(8 * g, a.dk - 8 - r0) * a.dv + min(l15, a.dv - 1 - col)),
                r0 + 8 * g < a.dk && col + l15 < a.dv, r0 < a.dk && col < a.dv};
    return {0, (unsigned)(min(row + 8 * g, a.dk - 1) * a.dv + min(col + l15, a.dv - 1)), row + 8 * g < a.dk && col + l15 < a.dv, true};
}
// f(t, j, r, base, at, in) for all a wave has that are live
template <int NKT, int NB, bool FAST, class F>
__device__ __forceinline__ void each_state(const nnsp_delta_args& a, int c0, int lane, const F& f) {
    const int l15 = lane & 15, g = lane >> 4;
    if (a.dk == 32 * NKT && c0 + 16 * NB <= a.dv) {
        const unsigned at = 8 * g * a.dv + l15;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int t = 0; t < 2 * NKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) f(t, j, r, (32 * (t >> 1) + 4 * (t & 1) + r) * a.dv + c0 + 16 * j, at, true);
    } else {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int t = 0; t < 2 * NKT; ++t) {
                if (!spot<FAST>(a, c0, t, j, 0, lane).live) continue;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const Spot p = spot<FAST>(a, c0, t, j, r, lane);
                    f(t, j, r, p.base, p.at, p.in);
                }
            }
    }
}

// A chunk's rows of q, k, g and beta of one stream and head: from global memory to
// registers, from there to LDS with what make_tp starts from.
template <class T, int NKT, int C, int PR, bool FAST>
struct Rows {
    const T *qp, *kp;
    const float *gp, *bp;
    long long qs, ks, gs, bs;
    RawRows<T, NKT, PR> rq, rk;
    float rg, rb;
    int row, part, lane, wave;

    // this thread's place in the chunk at frame t0
    __device__ __forceinline__ Rows(const nnsp_delta_args& a, int s, int h, long long t0, int tid, int wv)
        : row(tid / PR), part(tid % PR), lane(tid & 63), wave(wv) {
        const int hk = h / (a.value_heads / a.key_heads);
        qp = (const T*)a.q + s * a.q_stride[0] + hk * a.q_stride[2] + (t0 + row) * a.q_stride[1] + part * 8;
        kp = (const T*)a.k + s * a.k_stride[0] + hk * a.k_stride[2] + (t0 + row) * a.k_stride[1] + part * 8;
        const long long t = t0 + (lane & (C - 1));
        gp = a.g ? a.g + s * a.g_stride[0] + h * a.g_stride[2] + t * a.g_stride[1] : nullptr;
        bp = a.beta + s * a.beta_stride[0] + h * a.beta_stride[2] + t * a.beta_stride[1];
        qs = C * a.q_stride[1], ks = C * a.k_stride[1], gs = C * a.g_stride[1], bs = C * a.beta_stride[1];
    }
    // left: live frames from the chunk's first on
    __device__ __forceinline__ void fetch(int dk, int left) {
        fetch_rows<FAST>(rk, kp, part, dk, row < left);
        fetch_rows<FAST>(rq, qp, part, dk, row < left);
        fetch_gates(left);
    }
    __device__ __forceinline__ void fetch_gates(int left) {
        rg = rb = 0.0f;
        if (wave == 0 && (lane & (C - 1)) < left) {
            if (gp) rg = *gp;
            rb = *bp;
        }
    }
    __device__ __forceinline__ void next() {
        qp += qs, kp += ks, bp += bs;
        if (gp) gp += gs;
    }
    // of a scaled row, to its length 1 or to what it was; v_rsq_f32 and v_sqrt_f32 are good to one unit
    static __device__ __forceinline__ float factor(const nnsp_delta_args& a, float inv, float ss) {
        if (!(inv > 0.0f)) return 0.0f;  // a row of zeros
        if (!a.l2norm) return inv;
        const float s = inverse2(inv), e = a.eps * s * s;  // eps in the row's scale
        return e < INFINITY ? __builtin_amdgcn_rsqf(ss + e) : inv * __builtin_amdgcn_rsqf(a.eps);
    }
    __device__ __forceinline__ void stage(const nnsp_delta_args& a, KQ<T, NKT, C>& X, TP<T, C>& Y, Make<C>& M) {
        constexpr int KP = KQ<T, NKT, C>::KP;
        float ss, inv = stage_rows<KP>(rk, X.K, row, part, ss), x = factor(a, inv, ss);
        if (part == 0) M.kx[row] = x, M.kn[row] = x * __builtin_amdgcn_sqrtf(ss);
        inv = stage_rows<KP>(rq, X.Q, row, part, ss);
        x = a.scale * factor(a, inv, ss);
        if (part == 0) M.qx[row] = x, M.qn[row] = fabsf(x) * __builtin_amdgcn_sqrtf(ss);
        stage_gates(Y, M);
    }
    __device__ __forceinline__ void stage_gates(TP<T, C>& Y, Make<C>& M) {
        if (wave == 0) {
            // running sum of g in 64 bits, in units of log2, kept as two floats: differences of near frames stay exact
            const double x = scan_sum<C>((double)decay_log(rg) * 1.4426950408889634, lane);
            const int i = lane & (C - 1);  // of a chunk of 32, both halves of the wave alike
            M.gh[i] = (float)x;
            M.gl[i] = (float)(x - (double)(float)x);
            Y.beta[i] = rb;
        }
    }
};

// The same for FR frames of 16 NB columns of v by one wave, and for out the other way.
template <class T, int NKT, int NB, bool FAST, int FR, int C>
struct Cols {
    static constexpr int LPR = 2 * NB, ROWS = 64 / LPR < FR ? 64 / LPR : FR, N = FR / ROWS, VS = Geo<T, NKT, NB>::VS;
    typedef typename Vec<T, 8>::raw V8;
    typedef typename Vec<T, 8>::type V8u;
    typedef V8 V8s __attribute__((aligned(8)));  // in LDS
    const T* vp;
    T* op;
    long long vs, os, vc, oc;
    int row, col, left;  // left: columns from this lane's first on
    V8 x[N];

    __device__ __forceinline__ Cols(const nnsp_delta_args& a, int s, int h, long long t0, int c0, int lane)
        : row(lane / LPR), col((lane % LPR) * 8), left(row < ROWS ? a.dv - c0 - col : 0) {
        vp = (const T*)a.v + s * a.v_stride[0] + h * a.v_stride[2] + (t0 + row) * a.v_stride[1] + c0 + col;
        op = (T*)a.out + s * a.out_stride[0] + h * a.out_stride[2] + (t0 + row) * a.out_stride[1] + c0 + col;
        vs = ROWS * a.v_stride[1], os = ROWS * a.out_stride[1];
        vc = (C - FR) * a.v_stride[1], oc = (C - FR) * a.out_stride[1];  // from a chunk's last frame here to the next's first
    }
    // frames: live frames from the first here on
    __device__ __forceinline__ void fetch(int frames) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = (T)0.0f;
            const bool live = row + ROWS * i < frames;
            if (FAST) {
                if (live && left > 0) x[i] = *reinterpret_cast<const V8u*>(vp);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (live && j < left) x[i][j] = vp[j];
            }
            vp += vs;
        }
        vp += vc;
    }
    __device__ __forceinline__ void stage(T (*V)[VS]) const {
        if (row < ROWS)
#pragma unroll
            for (int i = 0; i < N; ++i) *reinterpret_cast<V8s*>(&V[row + ROWS * i][col]) = x[i];
        // the wave's own columns: LDS keeps its order within a wave, the compiler has to
        asm volatile("" ::: "memory");
    }
    __device__ __forceinline__ void store(T (*V)[VS], int frames) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool live = row < ROWS && row + ROWS * i < frames;
            if (FAST) {
                if (live && left > 0) *reinterpret_cast<V8u*>(op) = *reinterpret_cast<const V8s*>(&V[row + ROWS * i][col]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (live && j < left) op[j] = V[row + ROWS * i][col + j];
            }
            op += os;
        }
        op += oc;
    }
};

__device__ __forceinline__ int frames_of(const nnsp_delta_args& a, int s) {
    return a.lens ? max(0, min(a.lens[s], a.n_frames)) : a.n_frames;
}

// What a chunk of 32 needs no state for, before its inverse, by NW waves: the tiles
// of A ((0,0), (1,0), (1,1)) and of P, and the factors, which the tiles take in
// put(), with all waves together in between.
template <class T, int NKT, int NW>
struct Tiles {
    f32x4 ta, tp;
    // the wave's tile of A and of P; 3 and above: none
    static __device__ __forceinline__ int at(int role) { return role; }
    static __device__ __forceinline__ int pt(int role) {
        return NW == 4 ? (role == 3 ? 1 : role == 1 ? 3 : role) : role >= 3 ? role - 3 : 3;
    }
    __device__ __forceinline__ void dots(const KQ<T, NKT, CF>& X, TP<T, CF>& Y, Make<CF>& M, int role, int lane) {
        constexpr int KP = KQ<T, NKT, CF>::KP;
        const int l15 = lane & 15, g = lane >> 4, i = at(role), p = pt(role);
        if (i < 3) ta = dot_tile<NKT, KP>(X.K, X.K, i > 0, i > 1, l15, g);
        if (p < 3) tp = dot_tile<NKT, KP>(X.K, X.Q, p > 1, p > 0, l15, g);
        if (role == 1) make_factors<NKT>(X, Y, M, 0, lane);
        if (role == NW - 1) make_factors<NKT>(X, Y, M, 1, lane);
        if (role == (NW == 4 ? 1 : 6)) make_factors<NKT>(X, Y, M, 2, lane);
    }
    __device__ __forceinline__ void put(TP<T, CF>& Y, const Make<CF>& M, TriA<CF>& A, int role, int lane) const {
        const int l15 = lane & 15, g = lane >> 4, i = at(role), p = pt(role);
        if (i < 3) put_a(M, A, ta, i > 0, i > 1, l15, g);
        if (p < 3) put_p(Y, M, tp, p > 0, p > 1, l15, g);
        if (p == 0) put_p(Y, M, tp, 0, 1, l15, g);
    }
};

// Waves per SIMD that the state and the operands leave registers and LDS for.  Keys
// of 97 to 128 in 16 bits by 16 columns spill 7 to 39 registers at three, which
// two would not; 512 streams of 100 frames, 4 heads, at three and two, us, bf16
// and fp16: 128 x 64 111 and 112, 107 and 106; 128 x 48 103 and 100, 100 and 94;
// 100 x 64 (keys read by elements) 189 and 206, 191 and 203.
template <class T, int NKT, int NB, int NW>
constexpr int fused_waves() {
    return Geo<T, NKT, NB>::WIDE && NKT > 4 && NW == 4 ? 1 : Geo<T, NKT, NB>::WIDE || NB == 2 || NKT > 4 ? 2 : 3;
}

// Many streams: a workgroup per stream, head and 16 NB NW columns goes through its
// chunks of 32 alone, and the workgroups of a CU fill each other's waits.
// FAST: dk and dv are multiples of 8.  SPARE: dv leaves the last of them waves
// without columns, which only help with the tiles and the inverse (512 streams of
// 100 frames, 4 heads of 72 x 72, bf16: 139 -> 121 us; where all have some, asking
// costs registers: 8192 streams of 64 x 64 518 -> 528, fp32 of 128 x 128 252 ->
// 255, bf16 of 96 x 128 147 -> 149, of 128 x 128 171 -> 169).
//
// 100 frames of 8192 streams, 2 heads of 64 x 64, fp16: 500 us, of which the bytes
// alone would take 257; the vector units issue 67 % of the time (splits, factors,
// addresses: some 660 instructions a wave and chunk, and 38 matrix ones), at three
// waves a SIMD.  512 streams of 4 heads of 128 x 128, bf16: 169 us, bytes 98.
template <class T, int NKT, int NB, int NW, bool FAST, bool SPARE>
__global__ __launch_bounds__(64 * NW, (fused_waves<T, NKT, NB, NW>())) void delta_chunk_kernel(const nnsp_delta_args a) {
    using G = Geo<T, NKT, NB>;
    struct Lds {
        KQ<T, NKT, CF> X;
        TP<T, CF> Y;
        Make<CF> M;
        TriA<CF> A;
        alignas(16) T V[NW][CF][G::VS];  // each wave's columns of v, then of out
    };
    __shared__ Lds L;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ncb = (a.dv + 16 * NB * NW - 1) / (16 * NB * NW);
    const int cb = blockIdx.x % ncb, h = (blockIdx.x / ncb) % a.value_heads, s = blockIdx.x / ncb / a.value_heads;
    const int n = frames_of(a, s);
    const int c0 = (cb * NW + wave) * 16 * NB;  // first column of this wave
    const long long so = ((long long)s * a.value_heads + h) * a.dk * a.dv;
    const bool live = !SPARE || c0 < a.dv, spare = SPARE && (cb + 1) * 16 * NB * NW - 16 * NB >= a.dv;  // the last wave has none
    // who does what of the tiles: another SIMD each workgroup, or a wave without columns the longest part
    const int role = (wave + (spare ? 1 : blockIdx.x)) & (NW - 1);

    f32x4 S[2 * NKT][NB];
    float sinv[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        sinv[j] = 1.0f;
#pragma unroll
        for (int t = 0; t < 2 * NKT; ++t) S[t][j] = f32x4{0, 0, 0, 0};
    }
    if (a.state_in && live) {
        const float* sp = a.state_in + so;
        each_state<NKT, NB, FAST>(a, c0, lane, [&](int t, int j, int r, int base, unsigned at, bool in) {
            const float x = (sp + base)[at];
            S[t][j][r] = in ? x : 0.0f;
        });
    }
    Rows<T, NKT, CF, 2 * NW, FAST> rows(a, s, h, 0, tid, wave);
    Cols<T, NKT, NB, FAST, CF, CF> cols(a, s, h, 0, c0, lane);
    if (n > 0) {
        rows.fetch(a.dk, n);
        if (live) cols.fetch(n);
    }
    wait_loads();
    for (int t0 = 0; t0 < n; t0 += CF) {
        const int left = n - t0, nt = left > 16 ? 2 : 1, ln = here(lane);
        rows.stage(a, L.X, L.Y, L.M);
        if (live) cols.stage(L.V[wave]);
        __syncthreads();
        Tiles<T, NKT, NW> tiles;
        tiles.dots(L.X, L.Y, L.M, role, ln);
        __syncthreads();
        tiles.put(L.Y, L.M, L.A, role, ln);
        __syncthreads();
        if (role == 0) make_t(L.Y, L.A, ln, [] {});
        Chunk<T, NKT, NB> c;
        if (live) c.first(L.X, L.Y, L.V[wave], S, sinv, ln, nt);
        if (left > CF) {
            rows.next();
            rows.fetch(a.dk, left - CF);
            if (live) cols.fetch(left - CF);
        }
        __syncthreads();
        if (live) c.second(L.X, L.Y, L.V[wave], S, sinv, ln, nt, [] {});
        wait_loads();
        if (live) cols.store(L.V[wave], left);
        __syncthreads();
    }
    if (a.state_out && live) {
        float* sq = a.state_out + so;
        each_state<NKT, NB, FAST>(a, c0, here(lane), [&](int t, int j, int r, int base, unsigned at, bool in) {
            if (in) (sq + base)[at] = S[t][j][r] * sinv[j];
        });
    }
}

// Few rows, some chunks: the same with the parts of a chunk's work beside each
// other.  While waves 0 .. 3, 16 columns each, take chunk c through the state,
// wave 8 inverts chunk c + 1 and waves 4 .. 7 stage chunk c + 2 and make its
// tiles.  All meet three times a period; only 4 .. 7 need that.  A chunk of 128
// rows of 128 x 128, bf16, takes 3.1 us, where one part after the other takes
// about 5.
template <class T, int NKT>
struct PipeLds {
    KQ<T, NKT, CF> X[3];
    TP<T, CF> Y[3];
    Make<CF> M;
    TriA<CF> A[2];
    alignas(16) T V[4][CF][Geo<T, NKT, 1>::VS];
};
template <class T, int NKT, bool FAST>
__global__ __launch_bounds__(576) void delta_pipe_kernel(const nnsp_delta_args a) {
    __shared__ PipeLds<T, NKT> L;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ncb = (a.dv + 63) / 64;
    const int cb = blockIdx.x % ncb, h = (blockIdx.x / ncb) % a.value_heads, s = blockIdx.x / ncb / a.value_heads;
    const int n = frames_of(a, s), periods = n > 0 ? (n + CF - 1) / CF + 2 : 0;
    const auto meet = [] { __syncthreads(); };
    if (wave == 8) {
        for (int p = 0, i = 2; p < periods; ++p, i = i < 2 ? i + 1 : 0) {
            if (p >= 1 && p + 1 < periods) make_t(L.Y[i], L.A[(p + 1) & 1], here(lane), meet);
            else meet();
            meet();
            meet();
        }
        return;
    }
    if (wave >= 4) {
        const int role = wave - 4;
        Rows<T, NKT, CF, 8, FAST> rows(a, s, h, 0, threadIdx.x & 255, role);
        if (n > 0) rows.fetch(a.dk, n);
        for (int p = 0, i = 0; p < periods; ++p, i = i < 2 ? i + 1 : 0) {
            const int left = n - p * CF, ln = here(lane);
            if (left <= 0) {
                meet();
                meet();
                meet();
                continue;
            }
            rows.stage(a, L.X[i], L.Y[i], L.M);
            if (left > CF) {
                rows.next();
                rows.fetch(a.dk, left - CF);
            }
            meet();
            Tiles<T, NKT, 4> tiles;
            tiles.dots(L.X[i], L.Y[i], L.M, role, ln);
            meet();
            tiles.put(L.Y[i], L.M, L.A[p & 1], role, ln);
            meet();
        }
        return;
    }
    const int c0 = (cb * 4 + wave) * 16;
    const long long so = ((long long)s * a.value_heads + h) * a.dk * a.dv;
    f32x4 S[2 * NKT][1];
    float sinv[1] = {1.0f};
#pragma unroll
    for (int t = 0; t < 2 * NKT; ++t) S[t][0] = f32x4{0, 0, 0, 0};
    Cols<T, NKT, 1, FAST, CF, CF> cols(a, s, h, 0, c0, lane);
    if (a.state_in) {
        const float* sp = a.state_in + so;
        each_state<NKT, 1, FAST>(a, c0, lane, [&](int t, int j, int r, int base, unsigned at, bool in) {
            const float x = (sp + base)[at];
            S[t][j][r] = in ? x : 0.0f;
        });
    }
    if (n > 0) {
        cols.fetch(n);
        for (int i = 0; i < 6; ++i) meet();  // two periods
    }
    wait_loads();
    for (int p = 2, i = 0; p < periods; ++p, i = i < 2 ? i + 1 : 0) {
        const int left = n - (p - 2) * CF, nt = left > 16 ? 2 : 1, ln = here(lane);
        cols.stage(L.V[wave]);
        Chunk<T, NKT, 1> c;
        c.first(L.X[i], L.Y[i], L.V[wave], S, sinv, ln, nt);
        if (left > CF) cols.fetch(left - CF);
        meet();
        c.second(L.X[i], L.Y[i], L.V[wave], S, sinv, ln, nt, meet);
        wait_loads();
        cols.store(L.V[wave], left);
        meet();
    }
    if (a.state_out) {
        float* sq = a.state_out + so;
        each_state<NKT, 1, FAST>(a, c0, here(lane), [&](int t, int j, int r, int base, unsigned at, bool in) {
            if (in) (sq + base)[at] = S[t][j][r] * sinv[j];
        });
    }
}

// Few streams, many frames: T and P of all chunks at once, one workgroup each
// (prepare), then a short chain through the chunks (scan).  A slab of chunks
// goes through both before the next, so that its images are read while the
// caches still have them.
struct Slab {
    char *kq, *tp;          // images: [stream][key head][chunk of the slab], [stream][value head][chunk]
    int first, chunks;      // the slab's first chunk and its number of chunks
    const float* state_in;  // the chain's state before and after (NULL: zeros, dropped)
    float* state_out;
};

template <class X>
__device__ __forceinline__ void copy_out(char* dst, const X& src, int tid) {
    static_assert(sizeof(X) % 16 == 0, "whole 16-byte pieces");
    for (int i = tid; i < (int)(sizeof(X) / 16); i += 256)
        reinterpret_cast<f32x4*>(dst)[i] = reinterpret_cast<const f32x4*>(&src)[i];
}

// One workgroup per stream, key head and chunk, for all the key head's value heads.
// 64 chunks of 16 key heads and 32 value heads, 128 wide, bf16: 41 us for 34 MB in
// and 97 MB out, that is 2.4 TB/s of stores, where a large copy's are 2.5 (workgroups
// that stay and fetch their next chunk beside the work on one took as long).
template <class T, int NKT, bool FAST>
__global__ __launch_bounds__(256, (sizeof(KQ<T, NKT, C>) > 48 * 1024 ? 1 : 2)) void delta_prepare_kernel(const nnsp_delta_args a, const Slab b) {
    struct Lds {
        KQ<T, NKT, C> X;
        Make<C> M;
        Diag<C> D;
        TP<T, C> Y;
        char tail[sizeof(TriA<C>) - 2 * sizeof(Tri<C>)];  // A takes T's place and this
    };
    __shared__ Lds L;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = blockIdx.x % b.chunks, hk = (blockIdx.x / b.chunks) % a.key_heads, s = blockIdx.x / b.chunks / a.key_heads;
    const int rep = a.value_heads / a.key_heads, h0 = hk * rep;
    const int t0 = (b.first + c) * C, left = frames_of(a, s) - t0;
    if (left <= 0) return;
    Rows<T, NKT, C, 4, FAST> rows(a, s, h0, t0, tid, wave);
    rows.fetch(a.dk, left);
    rows.stage(a, L.X, L.Y, L.M);
    __syncthreads();
    copy_out(b.kq + (((long long)s * a.key_heads + hk) * b.chunks + c) * sizeof(KQ<T, NKT, C>), L.X, tid);
    for (int r = 0; r < rep; ++r) {
        if (r + 1 < rep) {
            if (rows.gp) rows.gp += a.g_stride[2];
            rows.bp += a.beta_stride[2];
            rows.fetch_gates(left);
        }
        make_tp(L.X, L.Y, L.M, L.D, *reinterpret_cast<TriA<C>*>(L.Y.T_), wave, here(lane));
        copy_out(b.tp + (((long long)s * a.value_heads + h0 + r) * b.chunks + c) * sizeof(TP<T, C>), L.Y, tid);
        if (r + 1 < rep) {
            __syncthreads();
            rows.stage_gates(L.Y, L.M);
            __syncthreads();
        }
    }
}

// Part `part` (0, 1, 2) of a chunk's two images into LDS past the registers, by
// waves `wave` of 4, 1 KB an instruction: a third each; of one buffer only for Y,
// half of X twice and then Y; of one buffer for both, all at the end.
template <int XB, int YB, class X, class Y>
__device__ __forceinline__ void copy_in(X& x, const char* sx, Y& y, const char* sy, int part, int wave, int lane) {
    constexpr int NX = sizeof(X) / 16, NY = sizeof(Y) / 16, BX = (NX + 63) / 64, BLOCKS = BX + (NY + 63) / 64;
    const auto bound = [](int p) { return p == 3 ? BLOCKS : YB == 2 ? BLOCKS * p / 3 : XB == 2 ? BX * p / 2 : 0; };
    for (int b = bound(part) + wave; b < bound(part + 1); b += 4) {
        const bool first = b < BX;
        const int i = (first ? b : b - BX) * 64;
        if (i + lane < (first ? NX : NY))
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)((first ? sx : sy) + (long long)(i + lane) * 16),
                (__attribute__((address_space(3))) void*)((first ? (char*)&x : (char*)&y) + i * 16), 16, 0, 0);
    }
}

// a tile times its rows' factors, as half of the high and low B operand that it is part of
__device__ __forceinline__ void put_part(h8 (*dst)[64], int lane, int half, const f32x4& x, const f32x4& s) {
    h4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = half_of(x[i], s[i]);
    reinterpret_cast<h4*>(&dst[0][lane])[half] = hi;
#pragma unroll
    for (int i = 0; i < 4; ++i) lo[i] = (_Float16)fmaf(x[i], s[i], -(float)hi[i]);
    reinterpret_cast<h4*>(&dst[1][lane])[half] = lo;
}

// What the four waves of a scan hand each other: B operands of 32 rows x 16
// columns, high and low, and each column's largest magnitudes of a wave, which
// set its scales.
template <int NKT, int NB>
struct Exchange {
    h8 S[NKT][NB][2][64], R[2][NB][2][64], U[2][NB][2][64], F[2][NB][2][64];  // S0, R, U for the output, U fk for the state
    float smax[NB][16][4], vmax[NB][16][4], fmax[NB][16][4];
};

// XB, YB: buffers of the two images
template <class T, int NKT, int NB, int XB, int YB>
struct ScanLds {
    KQ<T, NKT, C> X[XB];
    TP<T, C> Y[YB];
    Exchange<NKT, NB> E;
    alignas(16) T V[4][16][Geo<T, NKT, NB>::VS];
};

// The chain through the chunks for 16 NB columns: about 2 us a chunk (128 x 128,
// bf16), bound by the latency of its three exchanges.  Its length counts, so
// each of waves 0 .. 3 does a quarter of every product: a tile of 16 frames in
// K S0, T R, Q S0 and P U, a quarter of the state's rows in K^T U, handing its
// results on through LDS (three barriers a chunk).  Waves 4 .. 7 bring the next
// chunk's images meanwhile, a third after each barrier: all at once they hold up
// the products' own reads of LDS (64 chunks of 128 x 128 bf16: 126 us, all after
// the first barrier 148, none 121).  Where LDS has no room for two of an image, it
// comes after the third barrier, when the one before has been read.
// A column's scales have to be the same for all four before anybody has seen all
// its values: they come from bounds (|R| <= bmax |v| + xmax |S|, |u| <= 64 2^30,
// |S1| <= all |S0| + BOUND64 |U fk|) over the column's magnitudes exchanged at the
// barriers, sums of their largest terms.
template <class T, int NKT, int NB, bool FAST, int XB, int YB>
__global__ __launch_bounds__(512) void delta_scan_kernel(const nnsp_delta_args a, const Slab b) {
    using G = Geo<T, NKT, NB>;
    constexpr int TPW = (2 * NKT + 3) / 4;  // state tiles of a wave
    __shared__ ScanLds<T, NKT, NB, XB, YB> L;
    const int lane_ = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // streams and key heads vary fastest: with a multiple of 8 of them, all workgroups that read an image are on one XCD
    const unsigned keys = (unsigned)a.n_streams * a.key_heads;
    const int rep = a.value_heads / a.key_heads, hk = blockIdx.x % a.key_heads, s = blockIdx.x % keys / a.key_heads;
    const int cb = blockIdx.x / keys / rep, h = hk * rep + blockIdx.x / keys % rep;
    const int n = min(frames_of(a, s) - b.first * C, b.chunks * C);  // frames in this slab
    if (wave >= 4) {
        const char* kq = b.kq + ((long long)s * a.key_heads + hk) * b.chunks * sizeof(KQ<T, NKT, C>);
        const char* tp = b.tp + ((long long)s * a.value_heads + h) * b.chunks * sizeof(TP<T, C>);
        const auto load = [&](int i, int part) {
            copy_in<XB, YB>(L.X[i & (XB - 1)], kq, L.Y[i & (YB - 1)], tp, part, wave - 4, lane_);
            if (part == 2) kq += sizeof(KQ<T, NKT, C>), tp += sizeof(TP<T, C>);
        };
        // bare barriers: __syncthreads() would wait for the copies, which only the next chunk's first barrier has to
        const auto barrier = [] {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        if (n > 0) load(0, 0), load(0, 1), load(0, 2);
        barrier();
        for (int t0 = 0, i = 1; t0 < n; t0 += C, i ^= 1) {
            const bool more = n - t0 > C;
            wait_loads();
            barrier();  // this chunk is here, and the one before done with its buffers
            if (more) load(i, 0);
            barrier();
            if (more) load(i, 1);
            barrier();  // nothing reads this chunk's images any more
            if (more) load(i, 2);
        }
        return;
    }
    const int c0 = cb * 16 * NB;
    const long long so = ((long long)s * a.value_heads + h) * a.dk * a.dv;
    const f32x4 zero = {0, 0, 0, 0};
    f32x4 S[TPW][NB];
    float sinv[NB], sbound[NB], m[NB];  // of this lane's columns; sbound: of |S|, the registers' values
    // of all four waves, from what each has put where this lane's columns are
    const auto put_max = [&](float (*p)[16][4], int lane) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const float x = max_xor16_32(m[n]);
            if (lane < 16) p[n][lane][wave] = x;
        }
    };
    const auto max4 = [](const float* p) {
        const f32x4 x = ld4(p);
        return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    };
    // f(i, j, r, place, in) for element r of this wave's tile (i, j), as each_state
    const auto own_state = [&](int lane, const auto& f) {
#pragma unroll
        for (int i = 0; i < TPW; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                if (!spot<FAST>(a, c0, wave * TPW + i, j, 0, lane).live) continue;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const Spot p = spot<FAST>(a, c0, wave * TPW + i, j, r, lane);
                    f(i, j, r, so + p.base + p.at, p.in);
                }
            }
    };
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        sinv[j] = 1.0f;
        m[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < TPW; ++i) S[i][j] = zero;
    }
    if (b.state_in)
        own_state(lane_, [&](int i, int j, int r, long long at, bool in) {
            const float x = b.state_in[at];
            S[i][j][r] = in ? x : 0.0f;
            m[j] = fmaxf(m[j], fabsf(S[i][j][r]));
        });
    put_max(L.E.smax, lane_);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NB; ++n) sbound[n] = max4(L.E.smax[n][lane_ & 15]);

    Cols<T, NKT, NB, FAST, 16, C> cols(a, s, h, (long long)b.first * C + 16 * wave, c0, lane_);
    if (n > 0) cols.fetch(n - 16 * wave);
    wait_loads();
    for (int t0 = 0, i = 0; t0 < n; t0 += C, i ^= 1) {
        const int lane = here(lane_), l15 = lane & 15, g = lane >> 4, left = n - t0;
        const KQ<T, NKT, C>& X = L.X[i & (XB - 1)];
        const TP<T, C>& Y = L.Y[i & (YB - 1)];
        Exchange<NKT, NB>& E = L.E;
        // 1: the state's parts, and what bounds R
        float inv[NB];
        f32x4 vt[NB];
        cols.stage(L.V[wave]);
#pragma unroll
        for (int n = 0; n < NB; ++n) vt[n] = tile_of<T>(L.V[wave], n, l15, g);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const float sc = scale_of(sbound[n], inv[n]);
            inv[n] *= sinv[n];
            m[n] = 0.0f;
#pragma unroll
            for (int j = 0; j < TPW; ++j) {
                const int t = wave * TPW + j;
                if (t >= 2 * NKT) continue;  // not a tile of the state; its registers are never handed on
                put_part(E.S[t >> 1][n], lane, t & 1, S[j][n], all4(sc));
                m[n] = amax4(m[n], S[j][n]);
            }
        }
        put_max(E.smax, lane);
#pragma unroll
        for (int n = 0; n < NB; ++n) m[n] = amax4(0.0f, vt[n]);
        put_max(E.vmax, lane);
        __syncthreads();
        // 2: R and Q S0 of this wave's frames
        float sreg[NB], smax[NB], sc[NB], rinv[NB];  // the registers' values, the true ones; the scale of R and its inverse
        const float shared = poison(Y.bmax) + poison(Y.xmax);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            sreg[n] = max4(E.smax[n][l15]);
            smax[n] = sreg[n] * sinv[n];
            const float vmax = max4(E.vmax[n][l15]), bad = shared + poison(sreg[n]) + poison(vmax);
            sc[n] = scale_of(Y.bmax * vmax + Y.xmax * smax[n], rinv[n]);
            rinv[n] += bad;
            inv[n] += bad;
        }
        f32x4 O[NB];
        {
            f32x4 x[NB];
#pragma unroll
            for (int s = 0; s < NKT; ++s) {
                const int c = 32 * s + 8 * g;
                const h8 k = *reinterpret_cast<const h8*>(&X.K[0][16 * wave + l15][c]);
                const h8 q = *reinterpret_cast<const h8*>(&X.Q[0][16 * wave + l15][c]);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const h8 hi = E.S[s][n][0][lane], lo = E.S[s][n][1][lane];
                    x[n] = mma(k, lo, mma(k, hi, s ? x[n] : zero));
                    O[n] = mma(q, lo, mma(q, hi, s ? O[n] : zero));
                    if (G::KP == 2) {
                        x[n] = mma(*reinterpret_cast<const h8*>(&X.K[G::KP - 1][16 * wave + l15][c]), hi, x[n]);
                        O[n] = mma(*reinterpret_cast<const h8*>(&X.Q[G::KP - 1][16 * wave + l15][c]), hi, O[n]);
                    }
                }
            }
            const f32x4 bt = ld4(&Y.beta[16 * wave + 4 * g]), fx = ld4(&Y.fx[16 * wave + 4 * g]);
            const f32x4 fq = ld4(&Y.fq[16 * wave + 4 * g]);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const f32x4 f = fx * -inv[n];
                f32x4 r = vt[n] * bt;
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = fmaf(f[e], x[n][e], r[e]);
                put_part(E.R[wave >> 1][n], lane, wave & 1, r, all4(sc[n]));
                O[n] *= fq * inv[n];
            }
        }
        if (left > C) cols.fetch(left - C - 16 * wave);
        // what the next steps take of the images and know of the scales (see advance()), before the waits
        const float tmax = max4(Y.ti), cinv = tmax * 0x1p22f, c = inverse2(cinv), all = Y.all, ti = Y.ti[wave];
        float zi, s1[NB], d[NB];
        const float z = scale_of(Y.fkmax, zi) * 0x1p-14f;
        f32x4 f[NB];
        {
            const f32x4 fk = ld4(&Y.fk[16 * wave + 4 * g]);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float li;
                const float low = scale_of(fmaxf(smax[n] * (all * 0x1p-13f), 0x1p-86f), li);
                s1[n] = fminf(c * z * sc[n], low);
                d[n] = all * s1[n] * sinv[n];
                f[n] = fk * (ti * (s1[n] * rinv[n]));
            }
        }
        h8 th[2], tl[2];
#pragma unroll
        for (int s = 0; s < 2; ++s)
            if (2 * s <= wave) th[s] = Y.T_[0].operand(wave, l15, s, g), tl[s] = Y.T_[1].operand(wave, l15, s, g);
        __syncthreads();
        // 3: U of this wave's frames
        h8 kt[TPW][2][G::KP], ph[2], pl[2];
        f32x4 pi;
        {
            f32x4 u[NB];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (2 * s > wave) continue;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const h8 hi = E.R[s][n][0][lane], lo = E.R[s][n][1][lane];
                    u[n] = mma(tl[s], hi, mma(th[s], lo, mma(th[s], hi, s ? u[n] : zero)));
                }
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                put_part(E.F[wave >> 1][n], lane, wave & 1, u[n], f[n]);
                put_part(E.U[wave >> 1][n], lane, wave & 1, u[n], all4(ti * c));
                m[n] = amax4(0.0f, u[n] * f[n]);
            }
            put_max(E.fmax, lane);
#pragma unroll
            for (int j = 0; j < TPW; ++j) {
                const int t = min(wave * TPW + j, 2 * NKT - 1);
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int part = 0; part < G::KP; ++part) {
                        const int rw = 32 * s + 4 * g + (l15 >> 2), col = 32 * (t >> 1) + 8 * (l15 & 3) + 4 * (t & 1);
                        const h4 x = __builtin_bit_cast(h4, read_tr(&X.K[part][rw][col]));
                        const h4 y = __builtin_bit_cast(h4, read_tr(&X.K[part][rw + 16][col]));
                        kt[j][s][part] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                    }
#pragma unroll
                for (int n = 0; n < NB; ++n) S[j][n] *= d[n];
            }
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (2 * s <= wave) {
                    ph[s] = Y.P_[0].operand(wave, l15, s, g);
                    pl[s] = Y.P_[1].operand(wave, l15, s, g);
                }
            pi = ld4(&Y.pi[16 * wave + 4 * g]);
        }
        __syncthreads();
        // 4: this wave's rows of the state, its frames of the output
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            sbound[n] = fmaf(d[n], sreg[n], KQ<T, NKT, C>::BOUND64 * max4(E.fmax[n][l15]));
            sinv[n] = inverse2(s1[n]);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const h8 hi = E.F[s][n][0][lane], lo = E.F[s][n][1][lane];
#pragma unroll
                for (int j = 0; j < TPW; ++j) {
                    S[j][n] = mma(kt[j][s][0], lo, mma(kt[j][s][0], hi, S[j][n]));
                    if (G::KP == 2) S[j][n] = mma(kt[j][s][G::KP - 1], hi, S[j][n]);
                }
            }
        {
            f32x4 o[NB];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (2 * s > wave) continue;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const h8 hi = E.U[s][n][0][lane];
                    o[n] = mma(pl[s], hi, mma(ph[s], E.U[s][n][1][lane], mma(ph[s], hi, s ? o[n] : zero)));
                }
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const f32x4 p = pi * (rinv[n] * cinv);
#pragma unroll
                for (int r = 0; r < 4; ++r) L.V[wave][4 * g + r][16 * n + l15] = (T)fmaf(o[n][r], p[r], O[n][r]);
            }
        }
        wait_loads();
        cols.store(L.V[wave], left - 16 * wave);
    }
    if (b.state_out)
        own_state(here(lane_), [&](int i, int j, int r, long long at, bool in) {
            if (in) b.state_out[at] = S[i][j][r] * sinv[j];
        });
}

// ---- launches ----
template <class T, int NKT, int NB, int NW, bool FAST>
void launch_fused(const nnsp_delta_args& a, hipStream_t st) {
    constexpr int COLS = 16 * NB * NW;
    const int blocks = (a.dv + COLS - 1) / COLS;
    const dim3 grid((unsigned)((long long)a.n_streams * a.value_heads * blocks)), block(64 * NW);
    if constexpr (NKT <= 6) {  // wider keys leave no registers to ask
        if (blocks * COLS - 16 * NB >= a.dv) {
            delta_chunk_kernel<T, NKT, NB, NW, FAST, true><<<grid, block, 0, st>>>(a);
            return;
        }
    }
    delta_chunk_kernel<T, NKT, NB, NW, FAST, false><<<grid, block, 0, st>>>(a);
}

template <class T, int NKT, bool FAST>
void launch_pipe(const nnsp_delta_args& a, hipStream_t st) {
    const long long grid = (long long)a.n_streams * a.value_heads * ((a.dv + 63) / 64);
    delta_pipe_kernel<T, NKT, FAST><<<dim3((unsigned)grid), dim3(576), 0, st>>>(a);
}

template <class T, int NKT>
DeltaSplit plan_split(const nnsp_delta_args& a) {
    DeltaSplit p;
    const long long rows = (long long)a.n_streams * a.value_heads;
    p.chunks = (a.n_frames + C - 1) / C;
    p.kq_bytes = (long long)a.n_streams * a.key_heads * sizeof(KQ<T, NKT, C>);  // a chunk of all streams
    p.tp_bytes = rows * sizeof(TP<T, C>);
    const long long per = p.kq_bytes + p.tp_bytes;
    const int most = (int)(per * p.chunks <= DELTA_SLAB_BYTES ? p.chunks : DELTA_SLAB_BYTES / per < 1 ? 1 : DELTA_SLAB_BYTES / per);
    const int slabs = (p.chunks + most - 1) / most;
    p.slab = (p.chunks + slabs - 1) / slabs;  // of equal size
    p.state_bytes = p.slab < p.chunks ? (rows * a.dk * a.dv * 4 + 15) / 16 * 16 : 0;
    return p;
}

template <class T, int NKT, int NB, bool FAST>
void launch_scan(const nnsp_delta_args& a, const Slab& b, hipStream_t st) {
    constexpr int LDS = 160 * 1024, YB = sizeof(ScanLds<T, NKT, NB, 2, 2>) <= LDS ? 2 : 1,
                  XB = sizeof(ScanLds<T, NKT, NB, 2, YB>) <= LDS ? 2 : 1;
    const long long grid = (long long)a.n_streams * a.value_heads * ((a.dv + 16 * NB - 1) / (16 * NB));
    delta_scan_kernel<T, NKT, NB, FAST, XB, YB><<<dim3((unsigned)grid), dim3(512), 0, st>>>(a, b);
}

template <class T, int NKT, bool FAST>
void launch_split(const nnsp_delta_args& a, hipStream_t st) {
    const DeltaSplit p = plan_split<T, NKT>(a);
    const long long rows = (long long)a.n_streams * a.value_heads;
    char* w = (char*)a.workspace;
    float* carry = (float*)w;
    Slab b;
    b.kq = w + p.state_bytes;
    b.tp = b.kq + p.kq_bytes * p.slab;
    for (b.first = 0; b.first < p.chunks; b.first += p.slab) {
        b.chunks = p.chunks - b.first < p.slab ? p.chunks - b.first : p.slab;
        b.state_in = b.first ? carry : a.state_in;
        b.state_out = b.first + b.chunks < p.chunks ? carry : a.state_out;
        delta_prepare_kernel<T, NKT, FAST>
            <<<dim3((unsigned)((long long)a.n_streams * a.key_heads * b.chunks)), dim3(256), 0, st>>>(a, b);
        // 16 columns a workgroup while each still has a CU to itself, else 32 (LDS has room for one workgroup): 1000
        // frames of 128 x 128, bf16, us, 32 rows 49 and 61, 40 rows 81 and 68
        if (rows * ((a.dv + 15) / 16) <= 256) launch_scan<T, NKT, 1, FAST>(a, b, st);
        else launch_scan<T, NKT, 2, FAST>(a, b, st);
    }
}

// f<NKT, FAST>() of this call's sizes: keys go in by 32 columns, padded to one of
// a few widths (512 streams of 100 frames, 4 heads of 192 x 128, bf16: padded to
// 192 256 us, to 256 307; one stream of 4000 frames, 8 heads of 160 x 128, in two
// passes 158 and 245)
template <class F>
auto with_sizes(const nnsp_delta_args& a, const F& f) {
    typedef std::integral_constant<int, 1> I1;
    typedef std::integral_constant<int, 2> I2;
    typedef std::integral_constant<int, 3> I3;
    typedef std::integral_constant<int, 4> I4;
    typedef std::integral_constant<int, 6> I6;
    typedef std::integral_constant<int, 8> I8;
    if ((a.dk | a.dv) & 7)
        return a.dk <= 64 ? f(I2(), std::false_type()) : a.dk <= 128 ? f(I4(), std::false_type()) : f(I8(), std::false_type());
    if (a.dk <= 32) return f(I1(), std::true_type());
    if (a.dk <= 64) return f(I2(), std::true_type());
    if (a.dk <= 96) return f(I3(), std::true_type());
    if (a.dk <= 128) return f(I4(), std::true_type());
    if (a.dk <= 192) return f(I6(), std::true_type());
    return f(I8(), std::true_type());
}

template <class T>
DeltaSplit chunk_plan(const nnsp_delta_args& a) {
    return with_sizes(a, [&](auto nkt, auto) { return plan_split<T, decltype(nkt)::value>(a); });
}

template <class T>
int launch_chunk(const nnsp_delta_args& a, int split, hipStream_t st) {
    with_sizes(a, [&](auto nkt, auto fast) {
        constexpr int NKT = decltype(nkt)::value;
        constexpr bool FAST = decltype(fast)::value;
        constexpr bool WIDE = Geo<T, NKT, 1>::WIDE;
        // the first pass has no room in LDS for an image of 64 fp32 frames wider than 128
        if constexpr (!WIDE || NKT <= 4) {
            if (split) {
                launch_split<T, NKT, FAST>(a, st);
                return 0;
            }
        }
        // Workgroups of 64 columns that work on three chunks at once (pipe, keys up to 128 wide) while each has a CU to
        // itself, else such as share a CU, of 128 columns where there are so many (fused).  260 frames, dk = dv, us, pipe
        // against fused, bf16: 64, 32 rows 27 and 39, 256 rows 31 and 40, 384 rows 54 and 50; 128, 32 rows 33 and 51 (by 64
        // columns), 128 rows 38 and 54, 192 rows 66 and 61; fp32: 64, 256 rows 33 and 44, 384 rows 60 and 56; 128, 128
        // rows 42 and 61, 192 rows 77 and 63.  20 frames, 64: 7 and 7; 128, 128 rows 10 and 11.
        const long long groups = (long long)a.n_streams * a.value_heads * ((a.dv + 63) / 64);
        if constexpr (NKT <= 4) {
            if (groups <= 256) {
                launch_pipe<T, NKT, FAST>(a, st);
                return 0;
            }
        }
        // Keys over 128 leave registers for 64 columns in 16 bits (512 rows of 256 x 256, 200 frames: 256 us, 128 columns
        // by 8 waves 276), and fp32 is faster by 64 while CUs are left over (64 streams of 8 frames, 8
        // heads of 256 x 256: 112 us by 64, by 128 80; one stream, 2000 frames 529 and 617)
        const bool narrow = a.dv <= 64 || (NKT > 4 && groups <= 256);
        if constexpr (WIDE) narrow ? launch_fused<T, NKT, 1, 4, FAST>(a, st) : launch_fused<T, NKT, 1, 8, FAST>(a, st);
        else if constexpr (NKT > 4) launch_fused<T, NKT, 1, 4, FAST>(a, st);
        else narrow ? launch_fused<T, NKT, 1, 4, FAST>(a, st) : launch_fused<T, NKT, 2, 4, FAST>(a, st);
        return 0;
    });
    return (int)hipGetLastError();
}

}  // namespace

#endif
