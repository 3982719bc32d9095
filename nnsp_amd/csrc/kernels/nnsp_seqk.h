/* nnsp_seqk.h -- host <-> kernel interface of the sequence operators
 * (include/nnsp_seq.h).  The launchers take arguments that nnsp_seq.c has
 * checked. */
#ifndef NNSP_SEQK_H
#define NNSP_SEQK_H
#include "../../../include/nnsp_seq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* largest head width of the delta rule and row length of the norms */
#define NNSP_DELTA_MAX_D 256
#define NNSP_NORM_MAX_DIM 16384

int nnspk_launch_delta_step(const nnsp_delta_args *a, void *stream);
/* split: in two passes over the workspace, of nnspk_delta_split_bytes_*() bytes
 * (not of fp32 with dk > 128) */
int nnspk_launch_delta_chunk_f32(const nnsp_delta_args *a, int split, void *stream);
int nnspk_launch_delta_chunk_bf16(const nnsp_delta_args *a, int split, void *stream);
int nnspk_launch_delta_chunk_f16(const nnsp_delta_args *a, int split, void *stream);
long long nnspk_delta_split_bytes_f32(const nnsp_delta_args *a);
long long nnspk_delta_split_bytes_bf16(const nnsp_delta_args *a);
long long nnspk_delta_split_bytes_f16(const nnsp_delta_args *a);
int nnspk_launch_norm(const nnsp_norm_args *a, void *stream);

/* 1: kernels on device `dev` can use p (its own device memory, pinned host or
 * managed memory), 0: they cannot */
int nnspk_ptr_usable(const void *p, int dev);
/* device of a stream (NULL: the current device) */
int nnspk_stream_device(void *stream, int *dev);

#ifdef __cplusplus
}
#endif
#endif
