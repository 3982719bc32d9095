/*
 * nnsp_seq.h -- operators of floating-point sequence layers on MI355X
 * (libnnsp_mi355x.so), beside the fixed-point LSTM and FC layers of
 * nnsp_api.h / nnsp_batch.h and in the same layout: S independent streams,
 * T frames of each per call, stream-major, every stream's state carried from
 * call to call.
 *
 *   nnsp_delta_exec_device   the gated delta rule: a recurrent layer whose
 *                            state is a matrix per head, for one frame or a
 *                            chunk of frames per call
 *   nnsp_norm_exec_device    what stands around a block: post-norm, gate,
 *                            residual scale, residual add and the next
 *                            block's pre-norm, in one pass
 *
 * Conventions (as in nnsp_batch.h): plain pointers and sizes, integer return
 * codes (0 = ok, < 0 = argument error, > 0 = HIP error; nnsp_strerror).  Every
 * data pointer is memory the current HIP device can reach (hipMalloc'ed on it,
 * or pinned host / managed memory); memory of another device and pageable host
 * memory are refused with NNSP_EINVAL.  `stream` is a hipStream_t of that
 * device (NULL: its default stream).  The calls only queue kernels on it: they
 * allocate nothing, wait for nothing, and can be captured into a HIP graph.
 * The arguments are read before the call returns; nothing is kept from one
 * call to the next.
 */
#ifndef NNSP_SEQ_H
#define NNSP_SEQ_H
#include <stddef.h>
#include <stdint.h>

#include "nnsp_batch.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define NNSP_F32 0
#define NNSP_BF16 1
#define NNSP_F16 2

/*
 * Gated delta rule.  Per stream and value head h, with the key head
 * h / (value_heads / key_heads), state S [dk][dv]:
 *
 *   k^_t = k_t / sqrt(|k_t|^2 + eps), q^_t the same    (l2norm != 0; else as given;
 *                                                       a row of zeros stays zeros)
 *   S'   = exp(g_t) S_{t-1}
 *   u_t  = beta_t (v_t - S'^T k^_t)
 *   S_t  = S' + k^_t u_t^T
 *   o_t  = scale * S_t^T q^_t
 *
 * q, k [S][T][key_heads][dk], v, out [S][T][value_heads][dv] in `dtype`;
 * g, beta [S][T][value_heads] float; state_in, state_out
 * [S][value_heads][dk][dv] float, contiguous.  *_stride are the strides of
 * stream, frame and head in elements (the last dimension is contiguous; input
 * strides may be 0 to repeat a value, output elements must not coincide).
 * Only natural alignment of each type is asked for.
 *
 * lens [S] int32 (NULL: every stream has n_frames): frames of each stream, cut
 * to 0 .. n_frames.  Frames behind a stream's length are neither read nor
 * written, whatever they hold; a stream of length 0 keeps its state.
 * g NULL: no decay (g = 0).  state_in NULL: zeros.  state_out NULL: the final
 * state is dropped; it may be state_in itself (not a part of it).  out must
 * not overlap an input, nor any state.
 * g is a logarithm of the decay, normally <= 0; -infinity clears the state.
 * The state, sums and exponentials are held in 32 bits or more.  Calls of more
 * than NNSP_DELTA_STEP_FRAMES frames may run in chunks of up to 64 on the matrix
 * cores, whose products take the state, what is made of it and fp32 q and k in 22
 * bits, each column of the state and of v under scales of its own.  Decays above
 * 1 (g > 0) cost such calls precision by their product over 64 frames (beyond
 * 2^20 none is left: take such frames in calls of NNSP_DELTA_STEP_FRAMES).
 * How many streams, heads and frames a call has decides which of its forms runs;
 * what the other streams and heads hold changes no bit of a result.
 *
 * A value that is not finite in frame t spreads, as the recurrence has it, to
 * the later frames of its stream and head, from v and the state to their own
 * column only; in chunks it may reach the other frames of the same 64
 * (64 n .. 64 n + 63), earlier ones too.
 *
 * workspace: nnsp_delta_workspace() bytes of device memory, 16-byte aligned,
 * used by this call only while its kernels run (one workspace per call in
 * flight: calls on different streams, and graphs that may run at the same
 * time, need one each).
 *
 * Limits: dk, dv 1 .. 256; value_heads a multiple of key_heads;
 * n_frames at most 2^30; n_streams * value_heads * ceil(dv / 16) below 2^24.
 */
#define NNSP_DELTA_STEP_FRAMES 2
typedef struct {
    int32_t dtype;
    int32_t n_streams, n_frames;      /* S, T (0: nothing but the state's copy) */
    int32_t key_heads, value_heads;
    int32_t dk, dv;
    int32_t l2norm;
    float scale, eps;
    int64_t q_stride[3], k_stride[3], v_stride[3], g_stride[3], beta_stride[3], out_stride[3];
    const void *q, *k, *v;
    const float *g, *beta;
    const int32_t *lens;
    const float *state_in;
    void *out;
    float *state_out;
    void *workspace;
    size_t workspace_bytes;
} nnsp_delta_args;

/* Strides of contiguous tensors into *a, from its sizes. */
int nnsp_delta_contiguous(nnsp_delta_args *a);
/* Workspace of a call with these sizes (pointers and strides are not read). */
int nnsp_delta_workspace(const nnsp_delta_args *a, size_t *bytes);
int nnsp_delta_exec_device(const nnsp_delta_args *a, void *stream);

/*
 * Norms around a block.  Per row x of `dim` elements:
 *
 *   h = post(x)                             none | rms | layer norm, times w_post, plus b_post
 *   h = h * act(gate)                       none | sigmoid(z) | z sigmoid(z)
 *   r = res_in + res_scale * col_scale * h  (res_in NULL: 0; col_scale NULL: 1)
 *   res_out = r                             (NULL: not written)
 *   y = pre(r)                              none | rms | layer norm, times w_pre, plus b_pre
 *
 *   rms(x)   = x / sqrt(mean(x^2) + eps)
 *   layer(x) = (x - mean) / sqrt(mean((x - mean)^2) + eps)
 *
 * Everything between the loads and the stores is in 32 bits: y is the norm of
 * r itself, not of its rounding in res_out.
 *
 * x, gate, y are in `dtype`, res_in and res_out in `res_dtype` (`dtype` or
 * NNSP_F32), the weights, biases and col_scale float [dim] (NULL: ones, zeros,
 * ones).  Rows are addressed as [rows][groups] (frames and heads, say): each
 * tensor's *_stride holds the strides of both in elements, the row itself is
 * contiguous.  Input strides may be 0, output elements must not coincide.
 * y may be x or gate, and res_out may be res_in, where both have the same
 * strides; y or res_out NULL are not written (not both).  Outputs otherwise
 * overlap nothing.
 *
 * Limits: dim 1 .. 16384; rows * groups below 2^31.
 */
#define NNSP_NORM_NONE 0
#define NNSP_NORM_RMS 1
#define NNSP_NORM_LAYER 2
#define NNSP_GATE_NONE 0
#define NNSP_GATE_SIGMOID 1
#define NNSP_GATE_SILU 2
typedef struct {
    int32_t dtype, res_dtype;
    int32_t post, act, pre;           /* NNSP_NORM_*, NNSP_GATE_*, NNSP_NORM_* */
    int32_t dim;
    int64_t rows;
    int32_t groups, pad0;
    float eps_post, eps_pre, res_scale, pad1;
    int64_t x_stride[2], gate_stride[2], res_in_stride[2], res_out_stride[2], y_stride[2];
    const void *x, *gate, *res_in;
    const float *w_post, *b_post, *col_scale, *w_pre, *b_pre;
    void *res_out, *y;
} nnsp_norm_args;

/* Strides of contiguous tensors into *a, from its sizes. */
int nnsp_norm_contiguous(nnsp_norm_args *a);
int nnsp_norm_exec_device(const nnsp_norm_args *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif
