// nnsp_seq.hip -- the gated delta rule frame by frame, the fused norms, and the
// runtime queries of their argument checks (include/nnsp_seq.h).
#include "nnsp_seq_dev.h"
#include "nnsp_seqk.h"

namespace {

// ---- gated delta rule, one frame after another ------------------------------
// Columns of the state are independent, so a wave takes 4 CL columns of one
// stream and head and keeps them in registers for all the call's frames: CL
// lanes side by side hold 4 columns each, and 64 / CL groups of them RK rows
// each.  The state's read and write (8 dk dv bytes per stream and head) are what
// a single frame costs; a wave issues its RK 16-byte loads per lane before
// anything else.
//
// With S the state before the frame, o = scale (d S^T q + (k . q) u): both
// products with S and the three scalar products are summed over the row groups
// together, one cross-lane reduction per frame.
//
// One frame of 8192 streams, 2 heads of 64 x 64: 102 us, 5.4 TB/s of states, q, k,
// v and out, what a large copy reaches; of 128 streams, 32 heads of 128 x 128: 103
// us, 5.2 TB/s.  A frame of one stream takes 6 us on the device, a launch's and
// three dependent loads' latency.
template <class T, int RK>
struct FrameRaw {
    T k[RK], q[RK], v[4];
    float g, beta;
};

// x[j + sh], 0 beyond x[3]
template <class T>
__device__ __forceinline__ void shifted(T (&x)[4], int sh) {
    if constexpr (sizeof(T) == 2) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        const t4 v = {x[0], x[1], x[2], x[3]};
        const t4 r = __builtin_bit_cast(t4, sh < 4 ? __builtin_bit_cast(unsigned long long, v) >> (16 * (sh & 3)) : 0ull);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = r[j];
    } else {
#pragma unroll
        for (int b = 1; b <= 4; b *= 2)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (sh & b || sh > 4) x[j] = j + b < 4 ? x[j + b] : (T)0.0f;
    }
}

// elements r0 .. r0 + RK - 1 of n, zeros beyond them
template <class T, int RK>
__device__ __forceinline__ void load_rows(T (&d)[RK], const T* p, int r0, int n) {
    if (RK % 4 == 0 && (n & 3) == 0) {
#pragma unroll
        for (int c = 0; c < RK; c += 4) {
            T x[4];
            load_raw(x, p + (unsigned)min(r0 + c, n - 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) d[c + j] = r0 + c < n ? x[j] : (T)0.0f;
        }
    } else if (n >= 4) {
#pragma unroll
        for (int c = 0; c < RK; c += 4) {
            T x[4];
            const int at = min(r0 + c, n - 4);
            load_raw(x, p + (unsigned)at);
            shifted(x, r0 + c - at);
#pragma unroll
            for (int j = 0; j < 4 && c + j < RK; ++j) d[c + j] = x[j];
        }
    } else {
#pragma unroll
        for (int c = 0; c < RK; ++c) {
            const T x = p[(unsigned)min(r0 + c, n - 1)];
            d[c] = r0 + c < n ? x : (T)0.0f;
        }
    }
}

// columns c0 .. c0 + 3 of n of the row at p + row (p the same for all lanes)
template <class T>
__device__ __forceinline__ void load_cols(T (&d)[4], const T* p, unsigned row, int c0, int n, bool vec) {
    if (vec) {
        load_raw(d, p + (row + c0));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = p[row + min(c0 + j, n - 1)];
    }
}

// FULL: dk is 64 / CL RK and dv a multiple of 4
template <class T, int RK, int CL, bool FULL>
__global__ __launch_bounds__(256) void delta_step_kernel(const nnsp_delta_args a) {
    static_assert(CL == 8 || CL == 4, "");
    const int lane = threadIdx.x & 63;
    const int ncb = (a.dv + 4 * CL - 1) / (4 * CL);
    // where the waves of a head share 128-byte lines of its state, a range of its own for each of the 8 XCDs, so that
    // they share an L2 as well (dk = dv = 72: 3.6 -> 4.0 TB/s; without such lines it costs 2 %)
    const bool ranges = a.dv > 4 * CL && a.dv % 32;
    const unsigned block = ranges ? (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3) : blockIdx.x;
    const unsigned unit = block * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= (unsigned)a.n_streams * a.value_heads * ncb) return;
    const int cb = unit % ncb, h = (unit / ncb) % a.value_heads, s = unit / ncb / a.value_heads;
    const int hk = h / (a.value_heads / a.key_heads);
    const int rg = CL == 8 ? lane >> 3 : (lane & 3) | (lane >> 4) << 2, cl = CL == 8 ? lane & 7 : (lane >> 2) & 3;
    const int r0 = rg * RK, own = cb * 4 * CL + cl * 4;
    // a wave that has 4 columns: lanes whose 4 go past the last take the last 4, the same as others of the wave
    const bool vv = FULL || a.dv - cb * 4 * CL >= 4;
    const int c0 = vv ? min(own, a.dv - 4) : own;

    const long long so = ((long long)s * a.value_heads + h) * a.dk * a.dv;
    float S[RK][4];
    if (a.state_in) {
        const float* p = a.state_in + so;
#pragma unroll
        for (int r = 0; r < RK; ++r) {
            float x[4];
            load_cols(x, FULL ? p + r * a.dv : p, (FULL ? r0 : min(r0 + r, a.dk - 1)) * a.dv, c0, a.dv, vv);
#pragma unroll
            for (int j = 0; j < 4; ++j) S[r][j] = FULL || r0 + r < a.dk ? x[j] : 0.0f;
        }
    } else {
#pragma unroll
        for (int r = 0; r < RK; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) S[r][j] = 0.0f;
    }
    const int n = a.lens ? max(0, min(a.lens[s], a.n_frames)) : a.n_frames;

    const T* qp = (const T*)a.q + s * a.q_stride[0] + hk * a.q_stride[2];
    const T* kp = (const T*)a.k + s * a.k_stride[0] + hk * a.k_stride[2];
    const T* vp = (const T*)a.v + s * a.v_stride[0] + h * a.v_stride[2];
    const float* gp = a.g ? a.g + s * a.g_stride[0] + h * a.g_stride[2] : nullptr;
    const float* bp = a.beta + s * a.beta_stride[0] + h * a.beta_stride[2];
    T* op = (T*)a.out + s * a.out_stride[0] + h * a.out_stride[2];

    FrameRaw<T, RK> raw;
    const auto fetch = [&](long long t) {
        load_rows(raw.k, kp + t * a.k_stride[1], r0, a.dk);
        load_rows(raw.q, qp + t * a.q_stride[1], r0, a.dk);
        load_cols(raw.v, vp + t * a.v_stride[1], 0, c0, a.dv, vv);
        raw.g = gp ? gp[t * a.g_stride[1]] : 0.0f;
        raw.beta = bp[t * a.beta_stride[1]];
    };
    if (n > 0) fetch(0);
    for (int t = 0; t < n; ++t) {
        float k[RK], q[RK], v[4];
#pragma unroll
        for (int r = 0; r < RK; ++r) k[r] = (float)raw.k[r], q[r] = (float)raw.q[r];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)raw.v[j];
        const float dec = expf(decay_log(raw.g)), beta = raw.beta;
        if (t + 1 < n) fetch(t + 1);

        float sk[4], sq[4], kk, qq, kq;
        const auto sums = [&] {
            kk = qq = kq = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) sk[j] = sq[j] = 0.0f;
#pragma unroll
            for (int r = 0; r < RK; ++r) {
                kk = fmaf(k[r], k[r], kk);
                qq = fmaf(q[r], q[r], qq);
                kq = fmaf(k[r], q[r], kq);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sk[j] = fmaf(S[r][j], k[r], sk[j]);
                    sq[j] = fmaf(S[r][j], q[r], sq[j]);
                }
            }
            const auto rows_sum = [](float x) { return add_xor32(add_xor16(CL == 8 ? add_xor8(x) : add_xor2(add_xor1(x)))); };
#pragma unroll
            for (int j = 0; j < 4; ++j) sk[j] = rows_sum(sk[j]), sq[j] = rows_sum(sq[j]);
            kq = rows_sum(kq);
            if (a.l2norm) kk = rows_sum(kk), qq = rows_sum(qq);
        };
        sums();
        float rk = 1.0f, rq = 1.0f;
        if (a.l2norm) {
            float ek = a.eps, eq = a.eps;
            // squares that left 32 bits (the same in all lanes): the row at another scale, which its norm takes out again
            const auto outside = [](float x) { return !(x > 0x1p-100f && x < 0x1p100f); };
            if (outside(kk + ek) || outside(qq + eq)) {
                const float fk = kk > 1.0f ? 0x1p-80f : 0x1p60f, fq = qq > 1.0f ? 0x1p-80f : 0x1p60f;
                const bool ok = outside(kk + ek), oq = outside(qq + eq);
                ek = ok ? ek * fk * fk : ek;
                eq = oq ? eq * fq * fq : eq;
#pragma unroll
                for (int r = 0; r < RK; ++r) k[r] = ok ? k[r] * fk : k[r], q[r] = oq ? q[r] * fq : q[r];
                sums();
            }
            // a row of zeros stays one, also with eps 0
            rk = kk + ek == 0.0f ? 0.0f : 1.0f / sqrtf(kk + ek);
            rq = qq + eq == 0.0f ? 0.0f : 1.0f / sqrtf(qq + eq);
        }
        float u[4], o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u[j] = beta * (v[j] - dec * (rk * sk[j]));
            o[j] = a.scale * (rq * (dec * sq[j] + (rk * kq) * u[j]));
            u[j] *= rk;
        }
#pragma unroll
        for (int r = 0; r < RK; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) S[r][j] = fmaf(k[r], u[j], dec * S[r][j]);
        if (rg == 0) {
            T* p = op + t * a.out_stride[1];
            if (vv) {
                if (own < a.dv) store_vec(p + (unsigned)c0, o);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c0 + j < a.dv) p[(unsigned)(c0 + j)] = (T)o[j];
            }
        }
    }
    if (a.state_out) {
        float* p = a.state_out + so;
#pragma unroll
        for (int r = 0; r < RK; ++r) {
            if (!FULL && r0 + r >= a.dk) continue;
            float* base = FULL ? p + r * a.dv : p;
            const unsigned row = (FULL ? r0 : r0 + r) * a.dv;
            if (vv) {
                if (own < a.dv) store_vec(base + (row + c0), S[r]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c0 + j < a.dv) base[row + c0 + j] = S[r][j];
            }
        }
    }
}

// N rows a lane at least, of the few counts there are kernels for
template <class T, int CL, int N>
bool launch_step_rows(const nnsp_delta_args& a, hipStream_t st) {
    if (a.dk > 64 / CL * N) return false;
    const long long units = (long long)a.n_streams * a.value_heads * ((a.dv + 4 * CL - 1) / (4 * CL));
    const dim3 grid((unsigned)((units + 31) / 32 * 8)), block(256);  // a multiple of the 8 XCDs
    if constexpr (N % 4 == 0 || N > 8)
        if (a.dk == 64 / CL * N && a.dv % 4 == 0) {
            delta_step_kernel<T, N, CL, true><<<grid, block, 0, st>>>(a);
            return true;
        }
    delta_step_kernel<T, N, CL, false><<<grid, block, 0, st>>>(a);
    return true;
}
// Groups of 8 lanes read a row of the state by whole 128-byte lines (dk = dv =
// 64: 4.6 TB/s, with groups of 4 4.1); above 128 rows groups of 4 halve the
// registers a lane holds (144: 3.9 TB/s, with groups of 8 2.9).
template <class T, int CL, int... N>
void launch_step_of(const nnsp_delta_args& a, hipStream_t st) {
    (void)(launch_step_rows<T, CL, N>(a, st) || ...);
}
template <class T>
void launch_step(const nnsp_delta_args& a, hipStream_t st) {
    if (a.dk <= 128) launch_step_of<T, 8, 1, 2, 3, 4, 5, 6, 8, 9, 10, 12, 14, 16>(a, st);
    else launch_step_of<T, 4, 9, 10, 12, 14, 16>(a, st);
}

// ---- norms around a block ---------------------------------------------------
// One pass: TPR threads hold a row in registers (NCH chunks of 8 elements a
// thread), so each input is read once and each output written once; the call
// is bound by those bytes, provided that a gate's exponential and reciprocal
// are the hardware's (with their exact forms the vector units were the bound).
// Rows up to 1536 elements take 8 .. 64 lanes of a wave and sum by lane permutes;
// longer ones a whole workgroup and one LDS exchange per sum (32768 rows, two
// layer norms, bf16, by waves against workgroups: 1383 elements 75 us against 89,
// 1664 101 against 99, 2048 110 against 101).  Several short rows a thread, for
// more loads in flight, were no faster: 262144 gated rows of 64 17 us, four a
// thread 20.
//
// 1638400 rows of 64, gated, bf16: 107 us, 5.9 TB/s; 8192 of 4096 with an fp32
// residual: 79 us, 5.1 TB/s; 16384 of 2048 in fp32, gated: 119 us, 5.6 TB/s; a
// large copy 4.9 to 5.4.  5000 layer norms of 1001 with gate, residual and
// biases, fp16: 12 us, 4.1 TB/s; one row of 1024 3 us, a launch's and its loads'
// latency.
//
// ROW_FULL: the row is 8 TPR NCH elements.  ROW_TAIL: the row ends within a
// thread's chunk; that chunk then starts at n - 8, and what it has of the
// elements before is kept out of the sums (and stored twice, the same).
// ROW_TINY: fewer than 8 elements.
enum { ROW_FULL, ROW_TAIL, ROW_TINY };

template <int MODE>
struct Place {
    int c, first, n;  // where the chunk is, its first element that counts, the row's length
    Place() = default;
    __device__ __forceinline__ Place(int chunk, int n_) : c(chunk * 8), first(0), n(n_) {
        if (MODE == ROW_TAIL) {
            c = min(chunk * 8, n - 8);
            first = min(chunk * 8 - c, 8);
        }
    }
    __device__ __forceinline__ bool counts(int j) const {
        return MODE == ROW_FULL || (MODE == ROW_TAIL ? j >= first : c + j < n);
    }
    template <class T>
    __device__ __forceinline__ typename Vec<T, 8>::raw load(const T* p) const {
        typename Vec<T, 8>::raw x;
        if (MODE == ROW_TINY) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = p[min(c + j, n - 1)];
        } else {
            x = *reinterpret_cast<const typename Vec<T, 8>::type*>(p + c);
        }
        return x;
    }
    template <class T>
    __device__ __forceinline__ void store(T* p, const float (&s)[8]) const {
        if (MODE == ROW_TINY) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < n) p[c + j] = (T)s[j];
        } else if (MODE == ROW_FULL || first < 8) {
            store_vec(p + c, s);
        }
    }
};

template <int TPR>
struct RowSum {
    float* lds;
    int slot = 0;
    __device__ float operator()(float x) {
        if (TPR <= 64) return lane_sum<(TPR < 64 ? TPR : 64)>(x);
        x = lane_sum<64>(x);
        float* p = lds + slot++ * (TPR / 64);  // a place of its own per sum: one barrier each
        if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = x;
        __syncthreads();
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) s += p[i];
        return s;
    }
};

// the parts of a row in this thread, normed; w and b: this thread's weights
template <int TPR, int NCH, int MODE>
__device__ __forceinline__ void norm_row(float (&h)[NCH][8], int kind, float eps, const float (&w)[NCH][8], const float* bias,
                                         const Place<MODE> (&at)[NCH], int n, RowSum<TPR>& sum) {
    const float inv_n = 1.0f / (float)n;
    if (kind == NNSP_NORM_LAYER) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) m += at[i].counts(j) ? h[i][j] : 0.0f;
        m = sum(m) * inv_n;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] -= m;
    }
    const auto square = [&] {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) v = at[i].counts(j) ? fmaf(h[i][j], h[i][j], v) : v;
        return fmaf(sum(v), inv_n, eps);
    };
    float v = square();
    // squares that left 32 bits: such rows of the wave (a longer row is the same in all its waves) at another scale, which
    // the norm takes out again
    const bool outside = !(v > 0x1p-100f && v < INFINITY);
    if (__any(outside)) {
        const float f = !outside ? 1.0f : v > 1.0f ? 0x1p-80f : 0x1p90f;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] *= f;
        eps = eps * f * f;
        v = square();
    }
    // v_rsq_f32 is good to one unit in the last place; a row whose variance and eps are both 0 is infinite times 0, as
    // its definition is
    const float r = __builtin_amdgcn_rsqf(v);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] *= r * w[i][j];
        if (bias) {
            const auto x = at[i].load(bias);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] += x[j];
        }
    }
}

// sigmoid(z); PRECISE: the rounding of z log2(e), which the exponential takes up, is put back (fp32 outputs show it)
template <bool PRECISE>
__device__ __forceinline__ float sigmoid(float z) {
    const float l2e = 1.44269504f, t = -z * l2e;
    float e = __builtin_amdgcn_exp2f(t);
    if (PRECISE && fabsf(t) < 126.0f) {
        const float low = fmaf(-z, l2e, -t) - z * 1.925963e-8f;  // what t lacks of -z log2(e)
        e = fmaf(e, low * 0.69314718f, e);
    }
    return __builtin_amdgcn_rcpf(1.0f + e);
}

template <class T, class R, int TPR, int NCH, int MODE>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_kernel(const nnsp_norm_args a) {
    constexpr int RPB = TPR > 256 ? 1 : 256 / TPR;  // rows of a workgroup at a time
    __shared__ float red[6 * (TPR > 64 ? TPR / 64 : 1)];  // of two norms: the mean, the squares, at most once more
    RowSum<TPR> sum{red};
    const int tid = threadIdx.x % TPR, n = a.dim;
    const unsigned rows = (unsigned)a.rows * (unsigned)a.groups;
    const unsigned row = (blockIdx.y * gridDim.x + blockIdx.x) * (unsigned)RPB + threadIdx.x / TPR;  // < 2^31 + 2^28
    Place<MODE> at[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) at[i] = Place<MODE>(i * TPR + tid, n);
    typename Vec<T, 8>::raw x[NCH], z[NCH];
    typename Vec<R, 8>::raw q[NCH];
    // rows past the last read the last again (and store nothing)
    const unsigned live = min(row, rows - 1);
    long long ro = live, ri = 0;
    if (a.groups > 1) ro = live / (unsigned)a.groups, ri = live % (unsigned)a.groups;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        x[i] = at[i].load((const T*)a.x + ro * a.x_stride[0] + ri * a.x_stride[1]);
        if (a.act != NNSP_GATE_NONE) z[i] = at[i].load((const T*)a.gate + ro * a.gate_stride[0] + ri * a.gate_stride[1]);
        if (a.res_in) q[i] = at[i].load((const R*)a.res_in + ro * a.res_in_stride[0] + ri * a.res_in_stride[1]);
    }
    float wp[NCH][8], wn[NCH][8];
    const auto weights = [&](float (&w)[NCH][8], const float* p) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            if (p) {
                const auto v = at[i].load(p);
#pragma unroll
                for (int j = 0; j < 8; ++j) w[i][j] = v[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[i][j] = 1.0f;
            }
        }
    };
    if (a.post != NNSP_NORM_NONE) weights(wp, a.w_post);
    if (a.pre != NNSP_NORM_NONE) weights(wn, a.w_pre);
    // in place and without a norm, nothing else keeps a wave's stores behind the others' loads of the same tail
    if (TPR > 64 && MODE == ROW_TAIL && a.post == NNSP_NORM_NONE) __syncthreads();

    float h[NCH][8];
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = (float)x[i][j];
    if (a.post != NNSP_NORM_NONE) norm_row<TPR, NCH, MODE>(h, a.post, a.eps_post, wp, a.b_post, at, n, sum);
    if (a.act != NNSP_GATE_NONE)
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float g = (float)z[i][j], s = sigmoid<sizeof(T) == 4>(g);
                h[i][j] *= a.act == NNSP_GATE_SILU ? g * s : s;
            }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        if (a.col_scale) {
            const auto c = at[i].load(a.col_scale);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] *= c[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = a.res_in ? fmaf(a.res_scale, h[i][j], (float)q[i][j]) : a.res_scale * h[i][j];
    }
    if (a.res_out && row < rows) {
        R* p = (R*)a.res_out + ro * a.res_out_stride[0] + ri * a.res_out_stride[1];
#pragma unroll
        for (int i = 0; i < NCH; ++i) at[i].store(p, h[i]);
    }
    if (a.y) {
        if (a.pre != NNSP_NORM_NONE) norm_row<TPR, NCH, MODE>(h, a.pre, a.eps_pre, wn, a.b_pre, at, n, sum);
        if (row < rows) {
            T* p = (T*)a.y + ro * a.y_stride[0] + ri * a.y_stride[1];
#pragma unroll
            for (int i = 0; i < NCH; ++i) at[i].store(p, h[i]);
        }
    }
}

template <class T, class R, int TPR, int NCH, int MODE>
void launch_norm_mode(const nnsp_norm_args& a, hipStream_t st) {
    constexpr int PER = TPR > 256 ? 1 : 256 / TPR;
    // a grid has at most 2^32 - 1 threads along x
    const long long groups = (a.rows * a.groups + PER - 1) / PER, x = groups < (1 << 21) ? groups : 1 << 21;
    const dim3 grid((unsigned)x, (unsigned)((groups + x - 1) / x));
    norm_kernel<T, R, TPR, NCH, MODE><<<grid, dim3(TPR > 256 ? TPR : 256), 0, st>>>(a);
}
template <class T, class R, int TPR, int NCH>
void launch_norm_as(const nnsp_norm_args& a, hipStream_t st) {
    if (a.dim == 8 * TPR * NCH) launch_norm_mode<T, R, TPR, NCH, ROW_FULL>(a, st);
    else launch_norm_mode<T, R, TPR, NCH, ROW_TAIL>(a, st);
}

template <class T, class R>
void launch_norm_t(nnsp_norm_args a, hipStream_t st) {
    // rows and groups as one dimension where every tensor has them so
    const auto joined = [&](const int64_t* s) { return s[0] == s[1] * a.groups; };
    if (a.groups > 1 && joined(a.x_stride) && (!a.act || joined(a.gate_stride)) && (!a.res_in || joined(a.res_in_stride)) &&
        (!a.res_out || joined(a.res_out_stride)) && (!a.y || joined(a.y_stride))) {
        for (int64_t* s : {a.x_stride, a.gate_stride, a.res_in_stride, a.res_out_stride, a.y_stride}) s[0] = s[1];
        a.rows *= a.groups;
        a.groups = 1;
    }
    const int nc = (a.dim + 7) / 8;  // chunks of 8 elements
    if (a.dim < 8) launch_norm_mode<T, R, 8, 1, ROW_TINY>(a, st);
    else if (nc <= 8) launch_norm_as<T, R, 8, 1>(a, st);
    else if (nc <= 16) launch_norm_as<T, R, 16, 1>(a, st);
    else if (nc <= 32) launch_norm_as<T, R, 32, 1>(a, st);
    else if (nc <= 64) launch_norm_as<T, R, 64, 1>(a, st);
    else if (nc <= 128) launch_norm_as<T, R, 64, 2>(a, st);
    else if (nc <= 192) launch_norm_as<T, R, 64, 3>(a, st);
    else if (nc <= 256) launch_norm_as<T, R, 256, 1>(a, st);
    else if (nc <= 512) launch_norm_as<T, R, 256, 2>(a, st);
    else if (nc <= 1024) launch_norm_as<T, R, 512, 2>(a, st);
    else launch_norm_as<T, R, 1024, 2>(a, st);
}

int ok(hipError_t e) { return e == hipSuccess ? 0 : (int)e; }

}  // namespace

extern "C" {

int nnspk_launch_delta_step(const nnsp_delta_args* a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    if (a->dtype == NNSP_BF16) launch_step<__bf16>(*a, st);
    else if (a->dtype == NNSP_F16) launch_step<_Float16>(*a, st);
    else launch_step<float>(*a, st);
    return ok(hipGetLastError());
}

int nnspk_launch_norm(const nnsp_norm_args* a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const bool wide = a->res_dtype == NNSP_F32;
    if (a->dtype == NNSP_F32) launch_norm_t<float, float>(*a, st);
    else if (a->dtype == NNSP_BF16) wide ? launch_norm_t<__bf16, float>(*a, st) : launch_norm_t<__bf16, __bf16>(*a, st);
    else wide ? launch_norm_t<_Float16, float>(*a, st) : launch_norm_t<_Float16, _Float16>(*a, st);
    return ok(hipGetLastError());
}

int nnspk_ptr_usable(const void* p, int dev) {
    hipPointerAttribute_t at;
    if (hipPointerGetAttributes(&at, p) != hipSuccess) {
        (void)hipGetLastError();  // pageable host memory: not an error of a later call
        return 0;
    }
    if (at.type == hipMemoryTypeDevice) return at.device == dev;
    return at.type == hipMemoryTypeHost || at.type == hipMemoryTypeManaged;
}

int nnspk_stream_device(void* stream, int* dev) {
    if (!stream) return ok(hipGetDevice(dev));
    hipDevice_t d;
    const hipError_t e = hipStreamGetDevice((hipStream_t)stream, &d);
    if (e == hipSuccess) *dev = (int)d;
    else (void)hipGetLastError();
    return ok(e);
}

}  // extern "C"
