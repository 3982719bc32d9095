/*
 * nnsp_seq.c -- argument checks and dispatch of the sequence operators
 * (include/nnsp_seq.h).  Everything a kernel takes for granted about sizes,
 * strides and pointers is checked here, before the launch.
 */
#include <math.h>
#include <string.h>

#include "nnsp_host.h"
#include "../kernels/nnsp_seqk.h"

/* Largest |stride| and extent taken, in elements: offsets stay far inside 63 bits. */
#define MAX_STRIDE ((int64_t)1 << 46)
#define MAX_EXTENT ((int64_t)1 << 48)

static int size_of(int dtype) { return dtype == NNSP_F32 ? 4 : 2; }

static int bad(const char *who, const char *what)
{
    nnsp_set_error("%s: %s", who, what);
    return NNSP_EINVAL;
}

/* The strides of an input: not negative, not beyond MAX_STRIDE, the last
 * element within MAX_EXTENT.  Of an output also: no two elements in the same
 * place, that is, sorted by stride each dimension steps over all that is
 * inside it. */
static int check_strides(const char *who, const char *name, const int64_t *st, const int64_t *n, int dims, int64_t row,
                         int output)
{
    double reach = (double)row;
    for (int i = 0; i < dims; ++i)
        if (n[i] == 0) return 0; /* no element */
    for (int i = 0; i < dims; ++i) {
        if (st[i] < 0 || st[i] > MAX_STRIDE) {
            nnsp_set_error("%s: %s stride %lld out of range", who, name, (long long)st[i]);
            return NNSP_EINVAL;
        }
        if (n[i] > 1) reach += (double)st[i] * (double)(n[i] - 1);
    }
    if (reach > (double)MAX_EXTENT) {
        nnsp_set_error("%s: %s reaches over more than 2^48 elements", who, name);
        return NNSP_EINVAL;
    }
    if (!output) return 0;
    int used[3] = {0, 0, 0};
    int64_t inside = row; /* elements up to the end of what the dimensions so far span */
    for (int k = 0; k < dims; ++k) {
        int at = -1;
        for (int i = 0; i < dims; ++i)
            if (!used[i] && n[i] > 1 && (at < 0 || st[i] < st[at])) at = i;
        if (at < 0) break;
        used[at] = 1;
        if (st[at] < inside) {
            nnsp_set_error("%s: elements of %s coincide (stride %lld inside %lld elements)", who, name,
                           (long long)st[at], (long long)inside);
            return NNSP_EINVAL;
        }
        inside += st[at] * (n[at] - 1);
    }
    return 0;
}

typedef struct {
    const char *name;
    const void *p;
    size_t align; /* 0: the call does not use it */
} ptr_arg;

/* The current device, after checking that the stream is one of its. */
static int check_stream(const char *who, void *stream, int *dev)
{
    int sd = -1, e = nnspk_get_device(dev);
    if (!e) e = nnspk_stream_device(stream, &sd);
    if (e) return e;
    if (sd != *dev) {
        nnsp_set_error("%s: the stream belongs to device %d, the current one is %d", who, sd, *dev);
        return NNSP_EINVAL;
    }
    return 0;
}

/* The pointers of a call: first what needs no device (not NULL, natural
 * alignment), then that the current device can reach each. */
static int check_ptrs(const char *who, const ptr_arg *arg, int n, void *stream)
{
    int dev = 0;
    for (int i = 0; i < n; ++i) {
        if (!arg[i].align) continue;
        if (!arg[i].p) {
            nnsp_set_error("%s: %s is NULL", who, arg[i].name);
            return NNSP_EINVAL;
        }
        if ((uintptr_t)arg[i].p % arg[i].align) {
            nnsp_set_error("%s: %s is not aligned to %zu bytes", who, arg[i].name, arg[i].align);
            return NNSP_EINVAL;
        }
    }
    const int e = check_stream(who, stream, &dev);
    if (e) return e;
    for (int i = 0; i < n; ++i)
        if (arg[i].align && !nnspk_ptr_usable(arg[i].p, dev)) {
            nnsp_set_error("%s: %s is not memory of device %d", who, arg[i].name, dev);
            return NNSP_EINVAL;
        }
    return 0;
}

#define TRY(x)             \
    do {                   \
        int _e = (x);      \
        if (_e) return _e; \
    } while (0)

/* ---- gated delta rule ---- */

static int delta_sizes(const nnsp_delta_args *a, const char *who)
{
    if (!a) return bad(who, "NULL arguments");
    if (a->dtype != NNSP_F32 && a->dtype != NNSP_BF16 && a->dtype != NNSP_F16) return bad(who, "unknown dtype");
    if (a->n_streams < 0 || a->n_frames < 0) return bad(who, "negative n_streams or n_frames");
    if (a->key_heads < 1 || a->value_heads < 1 || a->value_heads % a->key_heads)
        return bad(who, "value_heads must be a positive multiple of key_heads");
    if (a->dk < 1 || a->dk > NNSP_DELTA_MAX_D || a->dv < 1 || a->dv > NNSP_DELTA_MAX_D) {
        nnsp_set_error("%s: dk, dv must be in 1..%d", who, NNSP_DELTA_MAX_D);
        return NNSP_EUNSUPPORTED;
    }
    if (a->n_frames > 1 << 30) {
        nnsp_set_error("%s: n_frames must be at most 2^30", who);
        return NNSP_EUNSUPPORTED;
    }
    if ((double)a->n_streams * a->value_heads * ((a->dv + 15) / 16) >= 16777216.0) { /* 256 threads each, 2^32 in all */
        nnsp_set_error("%s: n_streams * value_heads * ceil(dv / 16) must stay below 2^24", who);
        return NNSP_EUNSUPPORTED;
    }
    return 0;
}

static void dense3(int64_t *st, int64_t frames, int64_t heads, int64_t d)
{
    st[2] = d;
    st[1] = heads * d;
    st[0] = frames * heads * d;
}

int nnsp_delta_contiguous(nnsp_delta_args *a)
{
    TRY(delta_sizes(a, "nnsp_delta_contiguous"));
    dense3(a->q_stride, a->n_frames, a->key_heads, a->dk);
    dense3(a->k_stride, a->n_frames, a->key_heads, a->dk);
    dense3(a->v_stride, a->n_frames, a->value_heads, a->dv);
    dense3(a->out_stride, a->n_frames, a->value_heads, a->dv);
    dense3(a->g_stride, a->n_frames, a->value_heads, 1);
    dense3(a->beta_stride, a->n_frames, a->value_heads, 1);
    return 0;
}

/* How a call runs: frame by frame, in chunks, or in chunks in two passes. */
enum { DELTA_STEP, DELTA_CHUNK, DELTA_SPLIT };

static int delta_way(const nnsp_delta_args *a)
{
    /* A frame by itself costs 0.9 to 2 us after the first, a chunk of up to 32
     * about 6 to 10 us whatever it holds; rows of dk = 32 cost little more frame
     * by frame.  Frames against a chunk, bf16, us, 4096 rows: dk = dv = 32, 8
     * frames 26 against 36; 64, 4 frames 39 against 43, 6 frames 47 against 43;
     * 96, 4 frames 81 against 78, 6 frames 98 against 80; 128, 2 frames 119
     * against 127, 4 frames 154 against 128.  One row, 4 frames: 32 6.2 against
     * 6.2, 64 8.6 against 6.5, 128 9.4 against 7.6. */
    if (a->n_frames <= (a->dk <= 32 ? 8 : a->dk <= 96 ? 4 : NNSP_DELTA_STEP_FRAMES)) return DELTA_STEP;
    /* Two passes shorten the chain of a call whose few rows leave CUs idle, and
     * move twice the bytes.  What counts is how many workgroups of 16 columns
     * the second pass has for 256 CUs.  Chunks against two passes, us.  bf16, dk =
     * dv = 64: 256 workgroups, 260 frames 28 against 25, 500 frames 45 against 33;
     * 512: 260 frames 28 against 38, 500 frames 46 against 46; 768: 1000 frames 86
     * against 147.  128: 256, 130 frames 20 against 20, 260 frames 33 against 25;
     * 512: 260 frames 33 against 36, 500 frames 55 against 43, 1000 frames 104
     * against 74; 1024: 1000 frames 106 against 156.  fp32, 128: 256, 260 frames
     * 38 against 38, 500 frames 64 against 49; 512: 500 frames 65 against 63.
     * Wider keys, whose chunks go one after the other, 160 x 128, bf16: 256, 130
     * frames 31 against 23; 512, 260 frames 54 against 49.  LDS has no room for 64
     * frames of fp32 wider than 128. */
    const long long groups = (long long)a->n_streams * a->value_heads * ((a->dv + 15) / 16);
    if (a->dtype == NNSP_F32 && a->dk > 128) return DELTA_CHUNK;
    const int wide = a->dk > 128, from = groups <= 256 ? (wide ? 128 : 256) : wide ? 256 : 400;
    return groups <= 512 && a->n_frames >= from ? DELTA_SPLIT : DELTA_CHUNK;
}

int nnsp_delta_workspace(const nnsp_delta_args *a, size_t *bytes)
{
    if (!bytes) return bad("nnsp_delta_workspace", "NULL arguments");
    *bytes = 0;
    TRY(delta_sizes(a, "nnsp_delta_workspace"));
    if (delta_way(a) != DELTA_SPLIT || a->n_streams == 0) return 0;
    *bytes = (size_t)(a->dtype == NNSP_BF16  ? nnspk_delta_split_bytes_bf16(a)
                      : a->dtype == NNSP_F16 ? nnspk_delta_split_bytes_f16(a)
                                             : nnspk_delta_split_bytes_f32(a));
    return 0;
}

int nnsp_delta_exec_device(const nnsp_delta_args *a, void *stream)
{
    static const char who[] = "nnsp_delta_exec_device";
    size_t need = 0;
    TRY(delta_sizes(a, who));
    if (!isfinite(a->scale) || !(a->eps >= 0.0f) || !isfinite(a->eps)) return bad(who, "scale and eps must be finite, eps >= 0");
    const int64_t kn[3] = {a->n_streams, a->n_frames, a->key_heads};
    const int64_t vn[3] = {a->n_streams, a->n_frames, a->value_heads};
    TRY(check_strides(who, "q", a->q_stride, kn, 3, a->dk, 0));
    TRY(check_strides(who, "k", a->k_stride, kn, 3, a->dk, 0));
    TRY(check_strides(who, "v", a->v_stride, vn, 3, a->dv, 0));
    TRY(check_strides(who, "beta", a->beta_stride, vn, 3, 1, 0));
    if (a->g) TRY(check_strides(who, "g", a->g_stride, vn, 3, 1, 0));
    TRY(check_strides(who, "out", a->out_stride, vn, 3, a->dv, 1));
    if (a->n_streams == 0 || (a->n_frames == 0 && (!a->state_out || a->state_out == a->state_in))) return 0;
    if (a->state_in && a->state_out && a->state_in != a->state_out) {
        const uintptr_t i = (uintptr_t)a->state_in, o = (uintptr_t)a->state_out;
        const uintptr_t n = (uintptr_t)4 * a->n_streams * a->value_heads * a->dk * a->dv;
        if (i < o + n && o < i + n) return bad(who, "state_out overlaps state_in without being it");
    }
    if (a->n_frames > 0 && (a->out == a->q || a->out == a->k || a->out == a->v)) return bad(who, "out must not be q, k or v");
    TRY(nnsp_delta_workspace(a, &need));
    if (need && a->workspace_bytes < need) {
        nnsp_set_error("%s: workspace of %zu bytes, %zu needed", who, a->workspace_bytes, need);
        return NNSP_EINVAL;
    }
    const size_t el = a->n_frames > 0 ? (size_t)size_of(a->dtype) : 0, f = a->n_frames > 0 ? 4 : 0;
    const ptr_arg arg[] = {{"q", a->q, el},
                           {"k", a->k, el},
                           {"v", a->v, el},
                           {"out", a->out, el},
                           {"beta", a->beta, f},
                           {"g", a->g, a->g ? f : 0},
                           {"lens", a->lens, a->lens ? 4 : 0}, /* read without frames too */
                           {"state_in", a->state_in, a->state_in ? 4 : 0},
                           {"state_out", a->state_out, a->state_out ? 4 : 0},
                           {"workspace", a->workspace, need ? 16 : 0}};
    TRY(check_ptrs(who, arg, (int)(sizeof arg / sizeof *arg), stream));
    const int way = delta_way(a), split = way == DELTA_SPLIT;
    if (way == DELTA_STEP) return nnspk_launch_delta_step(a, stream);
    if (a->dtype == NNSP_BF16) return nnspk_launch_delta_chunk_bf16(a, split, stream);
    if (a->dtype == NNSP_F16) return nnspk_launch_delta_chunk_f16(a, split, stream);
    return nnspk_launch_delta_chunk_f32(a, split, stream);
}

/* ---- norms around a block ---- */

static int norm_sizes(const nnsp_norm_args *a, const char *who)
{
    if (!a) return bad(who, "NULL arguments");
    if (a->dtype != NNSP_F32 && a->dtype != NNSP_BF16 && a->dtype != NNSP_F16) return bad(who, "unknown dtype");
    if (a->res_dtype != NNSP_F32 && a->res_dtype != a->dtype) return bad(who, "res_dtype must be dtype or NNSP_F32");
    if (a->post < 0 || a->post > NNSP_NORM_LAYER || a->pre < 0 || a->pre > NNSP_NORM_LAYER) return bad(who, "unknown norm");
    if (a->act < 0 || a->act > NNSP_GATE_SILU) return bad(who, "unknown gate");
    if (a->dim < 1 || a->dim > NNSP_NORM_MAX_DIM) {
        nnsp_set_error("%s: dim must be in 1..%d", who, NNSP_NORM_MAX_DIM);
        return NNSP_EUNSUPPORTED;
    }
    if (a->rows < 0 || a->groups < 1) return bad(who, "rows must be >= 0, groups >= 1");
    if (a->rows > 2147483647 || (double)a->rows * a->groups >= 2147483648.0) {
        nnsp_set_error("%s: rows * groups must stay below 2^31", who);
        return NNSP_EUNSUPPORTED;
    }
    return 0;
}

int nnsp_norm_contiguous(nnsp_norm_args *a)
{
    TRY(norm_sizes(a, "nnsp_norm_contiguous"));
    int64_t *const st[5] = {a->x_stride, a->gate_stride, a->res_in_stride, a->res_out_stride, a->y_stride};
    for (int i = 0; i < 5; ++i) {
        st[i][0] = (int64_t)a->groups * a->dim;
        st[i][1] = a->dim;
    }
    return 0;
}

int nnsp_norm_exec_device(const nnsp_norm_args *a, void *stream)
{
    static const char who[] = "nnsp_norm_exec_device";
    TRY(norm_sizes(a, who));
    if (!(a->eps_post >= 0.0f) || !(a->eps_pre >= 0.0f) || !isfinite(a->eps_post) || !isfinite(a->eps_pre) ||
        !isfinite(a->res_scale))
        return bad(who, "eps and res_scale must be finite, eps >= 0");
    if (!a->y && !a->res_out) return bad(who, "y and res_out are both NULL");
    const int64_t n[2] = {a->rows, a->groups};
    TRY(check_strides(who, "x", a->x_stride, n, 2, a->dim, 0));
    if (a->act) TRY(check_strides(who, "gate", a->gate_stride, n, 2, a->dim, 0));
    if (a->res_in) TRY(check_strides(who, "res_in", a->res_in_stride, n, 2, a->dim, 0));
    if (a->res_out) TRY(check_strides(who, "res_out", a->res_out_stride, n, 2, a->dim, 1));
    if (a->y) TRY(check_strides(who, "y", a->y_stride, n, 2, a->dim, 1));
    if (a->y && ((a->y == a->x && memcmp(a->y_stride, a->x_stride, sizeof a->y_stride)) ||
                 (a->act && a->y == a->gate && memcmp(a->y_stride, a->gate_stride, sizeof a->y_stride))))
        return bad(who, "y in place of x or gate needs its strides");
    if (a->res_out && a->res_out == a->res_in && memcmp(a->res_out_stride, a->res_in_stride, sizeof a->res_out_stride))
        return bad(who, "res_out in place of res_in needs its strides");
    if (a->y && (a->y == a->res_in || a->y == a->res_out)) return bad(who, "y must not be res_in or res_out");
    if (a->res_out && (a->res_out == a->x || (a->act && a->res_out == a->gate)))
        return bad(who, "res_out must not be x or gate");
    if (a->rows == 0) return 0;
    const size_t el = (size_t)size_of(a->dtype), rl = (size_t)size_of(a->res_dtype);
    const ptr_arg arg[] = {{"x", a->x, el},
                           {"gate", a->gate, a->act ? el : 0},
                           {"res_in", a->res_in, a->res_in ? rl : 0},
                           {"res_out", a->res_out, a->res_out ? rl : 0},
                           {"y", a->y, a->y ? el : 0},
                           {"w_post", a->w_post, a->w_post ? 4 : 0},
                           {"b_post", a->b_post, a->b_post ? 4 : 0},
                           {"col_scale", a->col_scale, a->col_scale ? 4 : 0},
                           {"w_pre", a->w_pre, a->w_pre ? 4 : 0},
                           {"b_pre", a->b_pre, a->b_pre ? 4 : 0}};
    TRY(check_ptrs(who, arg, (int)(sizeof arg / sizeof *arg), stream));
    return nnspk_launch_norm(a, stream);
}
