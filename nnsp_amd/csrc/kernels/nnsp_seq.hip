// nnsp_seq.hip -- the gated delta rule frame by frame, the fused norms, and the
// runtime queries of their argument checks (include/nnsp_seq.h).
#include "nnsp_seq_dev.h"
#include "nnsp_seqk.h"

namespace {

// ---- gated delta rule, one frame after another ------------------------------
// Columns of the state are independent, so a wave takes 32 columns of one
// stream and head and keeps them in registers for all the call's frames: lane
// (rg, cl) = (lane / 8, lane % 8) holds rows rg * RK .. rg * RK + RK - 1 of
// columns 4 cl .. 4 cl + 3.  The state's read and write (8 dk dv bytes per
// stream and head) are what a single frame costs; a wave issues its RK 16-byte
// loads per lane (128-byte lines) before anything else.
//
// With S the state before the frame, o = scale (d S^T q + (k . q) u): both
// products with S and the three scalar products are summed over the row groups
// together, one cross-lane reduction per frame.
template <class T, int RK>
struct FrameRaw {
    T k[RK], q[RK], v[4];
    float g, beta;
};

template <class T, int RK>
__device__ __forceinline__ void load_rows(T (&d)[RK], const T* p, int r0, int n, bool vec) {
    if (vec) {
#pragma unroll
        for (int c = 0; c < RK; c += 4) {
            T x[4];
            load_raw(x, p + min(r0 + c, n - 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) d[c + j] = r0 + c < n ? x[j] : (T)0.0f;
        }
    } else {
#pragma unroll
        for (int c = 0; c < RK; ++c) {
            const T x = p[min(r0 + c, n - 1)];
            d[c] = r0 + c < n ? x : (T)0.0f;
        }
    }
}

template <class T>
__device__ __forceinline__ void load_cols(T (&d)[4], const T* p, int c0, int n, bool vec) {
    if (vec) {
        load_raw(d, p + min(c0, n - 4));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = p[min(c0 + j, n - 1)];
    }
}

template <class T, int RK>
__global__ __launch_bounds__(256) void delta_step_kernel(const nnsp_delta_args a) {
    const int lane = threadIdx.x & 63;
    const int ncb = (a.dv + 31) >> 5;
    const unsigned unit = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (unit >= (unsigned)a.n_streams * a.value_heads * ncb) return;
    const int cb = unit % ncb, h = (unit / ncb) % a.value_heads, s = unit / ncb / a.value_heads;
    const int hk = h / (a.value_heads / a.key_heads);
    const int r0 = (lane >> 3) * RK, c0 = cb * 32 + (lane & 7) * 4;
    const bool vk = (a.dk & 3) == 0, vv = (a.dv & 3) == 0;

    const long long so = ((long long)s * a.value_heads + h) * a.dk * a.dv;
    float S[RK][4];
    if (a.state_in) {
        const float* p = a.state_in + so;
#pragma unroll
        for (int r = 0; r < RK; ++r) {
            float x[4];
            load_cols(x, p + (long long)min(r0 + r, a.dk - 1) * a.dv, c0, a.dv, vv);
#pragma unroll
            for (int j = 0; j < 4; ++j) S[r][j] = r0 + r < a.dk ? x[j] : 0.0f;
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
    T* op = (T*)a.out + s * a.out_stride[0] + h * a.out_stride[2] + c0;

    FrameRaw<T, RK> raw;
    const auto fetch = [&](long long t) {
        load_rows(raw.k, kp + t * a.k_stride[1], r0, a.dk, vk);
        load_rows(raw.q, qp + t * a.q_stride[1], r0, a.dk, vk);
        load_cols(raw.v, vp + t * a.v_stride[1], c0, a.dv, vv);
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

        float sk[4] = {0, 0, 0, 0}, sq[4] = {0, 0, 0, 0}, kk = 0, qq = 0, kq = 0;
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
        const auto sum8 = [](float x) { return add_xor32(add_xor16(add_xor8(x))); };
#pragma unroll
        for (int j = 0; j < 4; ++j) sk[j] = sum8(sk[j]), sq[j] = sum8(sq[j]);
        kq = sum8(kq);
        float rk = 1.0f, rq = 1.0f;
        if (a.l2norm) {
            rk = 1.0f / sqrtf(sum8(kk) + a.eps);
            rq = 1.0f / sqrtf(sum8(qq) + a.eps);
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
        if (lane < 8) {
            T* p = op + t * a.out_stride[1];
            if (vv) {
                if (c0 < a.dv) store_vec(p, o);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c0 + j < a.dv) p[j] = (T)o[j];
            }
        }
    }
    if (a.state_out) {
        float* p = a.state_out + so + c0;
#pragma unroll
        for (int r = 0; r < RK; ++r) {
            if (r0 + r >= a.dk) continue;
            float* row = p + (long long)(r0 + r) * a.dv;
            if (vv) {
                if (c0 < a.dv) store_vec(row, S[r]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c0 + j < a.dv) row[j] = S[r][j];
            }
        }
    }
}

template <class T>
void launch_step(const nnsp_delta_args& a, hipStream_t st) {
    const long long units = (long long)a.n_streams * a.value_heads * ((a.dv + 31) / 32);
    const dim3 grid((unsigned)((units + 3) / 4)), block(256);
    const int rk = (a.dk + 7) / 8;
    if (rk <= 4) delta_step_kernel<T, 4><<<grid, block, 0, st>>>(a);
    else if (rk <= 8) delta_step_kernel<T, 8><<<grid, block, 0, st>>>(a);
    else if (rk <= 12) delta_step_kernel<T, 12><<<grid, block, 0, st>>>(a);
    else if (rk <= 16) delta_step_kernel<T, 16><<<grid, block, 0, st>>>(a);
    else if (rk <= 24) delta_step_kernel<T, 24><<<grid, block, 0, st>>>(a);
    else delta_step_kernel<T, 32><<<grid, block, 0, st>>>(a);
}

// ---- norms around a block ---------------------------------------------------
// One pass: TPR threads hold a row in registers (NCH chunks of 8 elements a
// thread), so each input is read once and each output written once; the call
// is bound by those bytes.  Rows up to 1024 elements take 8 .. 64 lanes of a
// wave and sum by lane permutes; longer ones a whole workgroup and one LDS
// exchange per sum.
template <class T>
__device__ __forceinline__ void load8(float (&d)[8], const T* p, int c, int n) {
    if (c + 8 <= n) {
        T x[8];
        load_raw(x, p + c);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = (float)x[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = c + j < n ? (float)p[c + j] : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&s)[8], int c, int n) {
    if (c + 8 <= n) {
        store_vec(p + c, s);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < n) p[c + j] = (T)s[j];
    }
}

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

template <int TPR, int NCH>
__device__ __forceinline__ void norm_row(float (&h)[NCH][8], int kind, float eps, const float* w, const float* b, int tid,
                                         int n, RowSum<TPR>& sum) {
    if (kind == NNSP_NORM_NONE) return;
    const float inv_n = 1.0f / (float)n;
    if (kind == NNSP_NORM_LAYER) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) m += h[i][j];
        m = sum(m) * inv_n;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = (i * TPR + tid) * 8 + j < n ? h[i][j] - m : 0.0f;
    }
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v = fmaf(h[i][j], h[i][j], v);
    const float r = 1.0f / sqrtf(sum(v) * inv_n + eps);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = (i * TPR + tid) * 8;
        float x[8];
        if (w) {
            load8(x, w, c, n);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] *= r * x[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] *= r;
        }
        if (b) {
            load8(x, b, c, n);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] += x[j];
        }
    }
}

template <class T, class R, int TPR, int NCH>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_kernel(const nnsp_norm_args a) {
    constexpr int RPB = TPR > 256 ? 1 : 256 / TPR;  // rows per workgroup
    __shared__ float red[4 * (TPR > 64 ? TPR / 64 : 1)];
    RowSum<TPR> sum{red};
    const int tid = threadIdx.x % TPR, n = a.dim;
    const long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
    if (row >= a.rows * a.groups) return;  // TPR > 64: one row per workgroup, all its threads together
    const long long ro = (unsigned)row / (unsigned)a.groups, ri = (unsigned)row % (unsigned)a.groups;
    const T* xp = (const T*)a.x + ro * a.x_stride[0] + ri * a.x_stride[1];
    const T* zp = (const T*)a.gate + ro * a.gate_stride[0] + ri * a.gate_stride[1];
    const R* rp = (const R*)a.res_in + ro * a.res_in_stride[0] + ri * a.res_in_stride[1];

    float h[NCH][8], z[NCH][8], r[NCH][8];
#pragma unroll
    for (int i = 0; i < NCH; ++i) load8(h[i], xp, (i * TPR + tid) * 8, n);
    if (a.act != NNSP_GATE_NONE)
#pragma unroll
        for (int i = 0; i < NCH; ++i) load8(z[i], zp, (i * TPR + tid) * 8, n);
    if (a.res_in) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) load8(r[i], rp, (i * TPR + tid) * 8, n);
    } else {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) r[i][j] = 0.0f;
    }

    norm_row<TPR, NCH>(h, a.post, a.eps_post, a.w_post, a.b_post, tid, n, sum);
    if (a.act != NNSP_GATE_NONE) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float g = 1.0f / (1.0f + expf(-z[i][j]));
                h[i][j] *= a.act == NNSP_GATE_SILU ? z[i][j] * g : g;
            }
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = (i * TPR + tid) * 8;
        if (a.col_scale) {
            float x[8];
            load8(x, a.col_scale, c, n);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] *= x[j];
        }
        // columns past the row's end hold 0 again (a bias or a gate of 0 may have moved them)
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = c + j < n ? fmaf(a.res_scale, h[i][j], r[i][j]) : 0.0f;
    }
    if (a.res_out) {
        R* p = (R*)a.res_out + ro * a.res_out_stride[0] + ri * a.res_out_stride[1];
#pragma unroll
        for (int i = 0; i < NCH; ++i) store8(p, h[i], (i * TPR + tid) * 8, n);
    }
    if (a.y) {
        norm_row<TPR, NCH>(h, a.pre, a.eps_pre, a.w_pre, a.b_pre, tid, n, sum);
        T* p = (T*)a.y + ro * a.y_stride[0] + ri * a.y_stride[1];
#pragma unroll
        for (int i = 0; i < NCH; ++i) store8(p, h[i], (i * TPR + tid) * 8, n);
    }
}

template <class T, class R, int TPR, int NCH>
void launch_norm_as(const nnsp_norm_args& a, hipStream_t st) {
    constexpr int RPB = TPR > 256 ? 1 : 256 / TPR;
    const long long rows = a.rows * a.groups;
    norm_kernel<T, R, TPR, NCH><<<dim3((unsigned)((rows + RPB - 1) / RPB)), dim3(TPR > 256 ? TPR : 256), 0, st>>>(a);
}

template <class T, class R>
void launch_norm_t(const nnsp_norm_args& a, hipStream_t st) {
    const int nc = (a.dim + 7) / 8;  // chunks of 8 elements
    if (nc <= 8) launch_norm_as<T, R, 8, 1>(a, st);
    else if (nc <= 16) launch_norm_as<T, R, 16, 1>(a, st);
    else if (nc <= 32) launch_norm_as<T, R, 32, 1>(a, st);
    else if (nc <= 64) launch_norm_as<T, R, 64, 1>(a, st);
    else if (nc <= 128) launch_norm_as<T, R, 64, 2>(a, st);
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
