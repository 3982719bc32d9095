"""Python host mirror of the sequence operators (include/nnsp_seq.h).

``GatedDelta`` is the gated delta rule, a recurrent layer with a matrix as each
head's state, for ``n_streams`` streams and up to ``n_frames`` frames of each per
call; ``BlockNorm`` is the post-norm, gate, residual scale and next pre-norm
around a block.  Both are plans: sizes, types and strides are fixed when they
are made, and every call takes device buffers as raw pointers (e.g.
``torch.Tensor.data_ptr()``) and queues its kernels on ``stream`` (a raw
``hipStream_t``, e.g. ``torch.cuda.current_stream().cuda_stream``; 0 or None:
the default stream).  The buffers have to live until the stream has passed them.
A plan is for one thread at a time; threads that call at once make one each.
"""
from __future__ import annotations

import ctypes as C
import struct

from . import _lib

DTYPES = {"f32": 0, "bf16": 1, "f16": 2}
NORMS = {"none": 0, "rms": 1, "layer": 2}
GATES = {"none": 0, "sigmoid": 1, "silu": 2}


def _one_of(table: dict, name: str, what: str) -> int:
    if name not in table:
        raise ValueError(f"{what} {name!r}: one of {', '.join(table)}")
    return table[name]


def _set(args, **numbers) -> None:
    """Integer fields of a struct, which ctypes alone would cut to their width."""
    for name, x in numbers.items():
        setattr(args, name, x)
        if getattr(args, name) != x:
            raise ValueError(f"{name} {x} is out of range")


def _set_strides(args, strides: dict | None, names: tuple, dims: int) -> None:
    for name, st in (strides or {}).items():
        if name not in names or len(st) != dims:
            raise ValueError(f"strides of {name!r}: {dims} numbers for one of {', '.join(names)}")
        st = [int(x) for x in st]
        getattr(args, name + "_stride")[:] = st
        if getattr(args, name + "_stride")[:] != st:
            raise ValueError(f"strides of {name!r} {st} are out of range")


def _packer(args, first: str, last: str):
    """pack(buffer, 0, ...) and the buffer of a struct's 8-byte fields first .. last: a call sets them all in one go."""
    begin, end = getattr(type(args), first).offset, getattr(type(args), last).offset + 8
    return (struct.Struct(f"{(end - begin) // 8}Q").pack_into,
            memoryview((C.c_char * (end - begin)).from_buffer(args, begin)))


class GatedDelta:
    """Plan of nnsp_delta_exec_device.

    ``scale`` defaults to dk ** -0.5.  ``strides``: {tensor: (stream, frame,
    head)} in elements for those of q, k, v, g, beta, out that are not
    contiguous [S][T][heads][d]."""

    def __init__(self, n_streams: int, n_frames: int, key_heads: int, value_heads: int, dk: int, dv: int,
                 dtype: str = "bf16", l2norm: bool = True, scale: float | None = None, eps: float = 1e-6,
                 strides: dict | None = None):
        a = self.args = _lib.DeltaArgs()
        a.dtype = _one_of(DTYPES, dtype, "dtype")
        _set(a, n_streams=n_streams, n_frames=n_frames, key_heads=key_heads, value_heads=value_heads, dk=dk, dv=dv)
        a.l2norm, a.eps = int(bool(l2norm)), eps
        L = _lib.lib()
        self._ref, self._call = C.byref(a), L.nnsp_delta_exec_device
        self._pack, self._ptrs = _packer(a, "q", "workspace_bytes")
        _lib.check(L.nnsp_delta_contiguous(self._ref), "nnsp_delta_contiguous")
        a.scale = dk ** -0.5 if scale is None else scale
        _set_strides(a, strides, ("q", "k", "v", "g", "beta", "out"), 3)
        n = C.c_size_t()
        _lib.check(L.nnsp_delta_workspace(self._ref, C.byref(n)), "nnsp_delta_workspace")
        self.workspace_bytes = n.value

    def exec_device(self, q: int, k: int, v: int, g: int | None, beta: int, out: int, state_in: int | None = None,
                    state_out: int | None = None, lens: int | None = None, workspace: int | None = None,
                    stream: int | None = None) -> None:
        """One call; ``workspace``: workspace_bytes bytes of device memory."""
        self._pack(self._ptrs, 0, q or 0, k or 0, v or 0, g or 0, beta or 0, lens or 0, state_in or 0, out or 0,
                   state_out or 0, workspace or 0, self.workspace_bytes if workspace else 0)
        rc = self._call(self._ref, stream)
        if rc:
            _lib.check(rc, "nnsp_delta_exec_device")


class BlockNorm:
    """Plan of nnsp_norm_exec_device for [rows][groups] rows of ``dim`` elements.

    ``strides``: {tensor: (row, group)} in elements for those of x, gate,
    res_in, res_out, y that are not contiguous [rows][groups][dim]."""

    def __init__(self, rows: int, dim: int, groups: int = 1, dtype: str = "bf16", res_dtype: str | None = None,
                 post: str = "rms", act: str = "none", pre: str = "rms", res_scale: float = 1.0, eps: float = 1e-6,
                 eps_post: float | None = None, strides: dict | None = None):
        a = self.args = _lib.NormArgs()
        a.dtype = _one_of(DTYPES, dtype, "dtype")
        a.res_dtype = a.dtype if res_dtype is None else _one_of(DTYPES, res_dtype, "res_dtype")
        a.post, a.pre = _one_of(NORMS, post, "post"), _one_of(NORMS, pre, "pre")
        a.act = _one_of(GATES, act, "act")
        _set(a, rows=rows, groups=groups, dim=dim)
        a.eps_pre, a.eps_post, a.res_scale = eps, eps if eps_post is None else eps_post, res_scale
        L = _lib.lib()
        self._ref, self._call = C.byref(a), L.nnsp_norm_exec_device
        self._pack, self._ptrs = _packer(a, "x", "y")
        _lib.check(L.nnsp_norm_contiguous(self._ref), "nnsp_norm_contiguous")
        _set_strides(a, strides, ("x", "gate", "res_in", "res_out", "y"), 2)

    def exec_device(self, x: int, y: int | None, gate: int | None = None, w_post: int | None = None,
                    b_post: int | None = None, col_scale: int | None = None, w_pre: int | None = None,
                    b_pre: int | None = None, res_in: int | None = None, res_out: int | None = None,
                    stream: int | None = None) -> None:
        self._pack(self._ptrs, 0, x or 0, gate or 0, res_in or 0, w_post or 0, b_post or 0, col_scale or 0, w_pre or 0,
                   b_pre or 0, res_out or 0, y or 0)
        rc = self._call(self._ref, stream)
        if rc:
            _lib.check(rc, "nnsp_norm_exec_device")
