"""Sequence operators (include/nnsp_seq.h), host side: the ctypes mirrors, the
exported symbols, and every refusal that needs no GPU."""
import ctypes as C
import os
import re
import subprocess
import threading

import pytest

from conftest import ROOT
from nnsp_amd import _lib
from nnsp_amd.seq import BlockNorm, GatedDelta

BAD = 3 << 12  # an aligned address that nothing is read from: these calls fail before any use


def test_declared_symbols_are_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "nnsp_seq.h")).read(), flags=re.S)
    names = set(re.findall(r"\bint (nnsp_\w+)\(", text))
    assert names == {"nnsp_delta_contiguous", "nnsp_delta_workspace", "nnsp_delta_exec_device",
                     "nnsp_norm_contiguous", "nnsp_norm_exec_device"}
    assert all(hasattr(_lib.lib(), n) for n in names)


@pytest.mark.parametrize("struct,mirror", [("nnsp_delta_args", _lib.DeltaArgs), ("nnsp_norm_args", _lib.NormArgs)])
def test_struct_mirrors(tmp_path, struct, mirror):
    fields = [f for f, _ in mirror._fields_]
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include "nnsp_seq.h"\nint main(void) {\n'
                   + f'printf("%zu\\n", sizeof({struct}));\n'
                   + "".join(f'printf("%zu\\n", offsetof({struct}, {f}));\n' for f in fields) + "return 0; }\n")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "p")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "p")]).split()]
    assert got == [C.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]


def refused(call, message, code=_lib.NNSP_EINVAL):
    with pytest.raises(RuntimeError, match=message) as e:
        call()
    assert f"error {code}:" in str(e.value)


@pytest.mark.parametrize("sizes,message,code", [
    ((-1, 1, 1, 1, 8, 8), "negative", -1), ((1, -1, 1, 1, 8, 8), "negative", -1),
    ((1, 1, 0, 1, 8, 8), "multiple of key_heads", -1), ((1, 1, 2, 3, 8, 8), "multiple of key_heads", -1),
    ((1, 1, 1, 0, 8, 8), "multiple of key_heads", -1),
    ((1, 1, 1, 1, 0, 8), "dk, dv", -2), ((1, 1, 1, 1, 257, 8), "dk, dv", -2), ((1, 1, 1, 1, 8, 257), "dk, dv", -2),
    ((1 << 30, 1, 1, 2, 8, 8), "below 2", -2),
    ((1 << 23, 1, 1, 1, 8, 17), "below 2", -2), ((1, (1 << 30) + 1, 1, 1, 8, 8), "n_frames", -2),
])
def test_delta_sizes_refused(sizes, message, code):
    refused(lambda: GatedDelta(*sizes), message, code)


@pytest.mark.parametrize("make", [
    lambda: GatedDelta((1 << 32) + 1, 1, 1, 1, 8, 8), lambda: GatedDelta(1, (1 << 32) + 3, 1, 1, 8, 8),
    lambda: GatedDelta(1, 1, 1, 1, 8, (1 << 32) + 8), lambda: BlockNorm(1, (1 << 32) + 8), lambda: BlockNorm((1 << 64) + 1, 8),
    lambda: BlockNorm(1, 8, groups=(1 << 32) + 1), lambda: BlockNorm(1, 8, strides={"x": ((1 << 64) + 8, 8)}),
    lambda: GatedDelta(1, 1, 1, 1, 8, 8, strides={"v": (8, 8, 1 << 64)}),
])
def test_sizes_beyond_their_fields_are_refused(make):
    with pytest.raises(ValueError, match="out of range"):
        make()


def test_delta_unknown_dtype():
    with pytest.raises(ValueError, match="one of"):
        GatedDelta(1, 1, 1, 1, 8, 8, dtype="f64")
    p = GatedDelta(1, 1, 1, 1, 8, 8)
    p.args.dtype = 7
    refused(lambda: p.exec_device(BAD, BAD, BAD, BAD, BAD, BAD + 4096), "unknown dtype")


def delta(call=None, strides=None, sizes=(2, 3, 1, 2, 8, 8), **kw):
    p = GatedDelta(*sizes, strides=strides, **kw)
    ptrs = dict(q=BAD, k=BAD, v=BAD, g=BAD, beta=BAD, out=BAD + 4096)
    ptrs.update(call or {})
    n = ptrs.pop("workspace_bytes", None)
    if n is not None:
        p.workspace_bytes = n
    return lambda: p.exec_device(**ptrs)


@pytest.mark.parametrize("call,message", [
    ({"q": None}, "q is NULL"), ({"k": None}, "k is NULL"), ({"v": None}, "v is NULL"), ({"beta": None}, "beta is NULL"),
    ({"out": None}, "out is NULL"), ({"q": BAD + 1}, "q is not aligned"), ({"g": BAD + 2}, "g is not aligned"),
    ({"state_in": BAD + 2}, "state_in is not aligned"), ({"state_out": BAD + 1}, "state_out is not aligned"),
    ({"lens": BAD + 2}, "lens is not aligned"), ({"out": BAD}, "out must not be"),
    ({"state_in": BAD, "state_out": BAD + 4}, "overlaps"), ({"state_in": BAD + 16, "state_out": BAD}, "overlaps"),
])
def test_delta_pointers_refused(call, message):
    refused(delta(call), message)


@pytest.mark.parametrize("strides,message", [
    ({"q": (-8, 8, 8)}, "q stride"), ({"k": (8, 1 << 47, 8)}, "k stride"),
    ({"out": (48, 16, 4)}, "coincide"), ({"out": (48, 0, 8)}, "coincide"), ({"out": (40, 16, 8)}, "coincide"),
    ({"v": (1 << 46, 1 << 45, 8)}, None),
])
def test_delta_strides_refused(strides, message):
    if message is None:  # within the limits: refused only for want of a device or of real memory
        with pytest.raises(RuntimeError) as e:
            delta({"v": None}, strides)()
        assert "v is NULL" in str(e.value)
    else:
        refused(delta(strides=strides), message)


def test_delta_strides_reach():
    st = {"v": (1 << 46, 8, 8)}
    refused(delta(strides=st, sizes=(9, 3, 1, 2, 8, 8)), "2\\^48")


def test_delta_names_of_strides():
    for st in ({"x": (1, 1, 1)}, {"q": (1, 1)}):
        with pytest.raises(ValueError, match="strides of"):
            GatedDelta(1, 1, 1, 1, 8, 8, strides=st)


@pytest.mark.parametrize("kw", [{"scale": float("inf")}, {"scale": float("nan")}, {"eps": -1.0}, {"eps": float("nan")}])
def test_delta_scalars_refused(kw):
    refused(delta(**kw), "finite")


def test_delta_workspace():
    """Few streams over many frames ask for one, bounded however long they are; others do not."""
    assert GatedDelta(1, 8, 1, 1, 64, 64).workspace_bytes == 0
    assert GatedDelta(8192, 100, 2, 2, 64, 64).workspace_bytes == 0
    assert GatedDelta(0, 1000, 2, 2, 64, 64).workspace_bytes == 0
    n = [GatedDelta(1, T, 16, 32, 128, 128).workspace_bytes for T in (256, 16384, 1 << 30)]
    assert 0 < n[0] < n[1] <= n[2] < 128 << 20
    refused(delta(sizes=(2, 1000, 1, 2, 64, 64)), "workspace of 0 bytes")
    refused(delta({"workspace": BAD + 8}, sizes=(2, 1000, 1, 2, 64, 64)), "workspace is not aligned")


def test_delta_nothing_to_do():
    delta(sizes=(0, 3, 1, 2, 8, 8))()
    delta({"q": None, "k": None, "v": None, "beta": None, "out": None}, sizes=(2, 0, 1, 2, 8, 8))()


def test_delta_lens_are_checked_without_frames_too():
    """The copy of the state still reads every stream's length."""
    refused(delta({"lens": BAD + 2, "state_in": BAD, "state_out": BAD + 4096}, sizes=(2, 0, 1, 2, 8, 8)), "lens is not aligned")


def test_refusals_keep_to_their_thread():
    """What one thread's call was refused for is not overwritten by another thread's refusal."""
    L = _lib.lib()
    plans = [GatedDelta(1, 1, 1, 1, 8, 8) for _ in range(2)]
    plans[0].args.out, plans[1].args.dtype = BAD, 7
    assert L.nnsp_delta_exec_device(plans[0]._ref, None) == _lib.NNSP_EINVAL
    mine = L.nnsp_strerror(_lib.NNSP_EINVAL)
    seen = []

    def other():
        seen.append(L.nnsp_strerror(_lib.NNSP_EINVAL))
        assert L.nnsp_delta_exec_device(plans[1]._ref, None) == _lib.NNSP_EINVAL
        seen.append(L.nnsp_strerror(_lib.NNSP_EINVAL))

    t = threading.Thread(target=other)
    t.start()
    t.join()
    assert b"q is NULL" in mine and L.nnsp_strerror(_lib.NNSP_EINVAL) == mine
    assert seen[0] == b"invalid argument" and b"unknown dtype" in seen[1]


def test_null_arguments():
    L = _lib.lib()
    n = C.c_size_t()
    assert L.nnsp_delta_exec_device(None, None) == _lib.NNSP_EINVAL
    assert L.nnsp_delta_workspace(None, C.byref(n)) == _lib.NNSP_EINVAL
    assert L.nnsp_delta_workspace(GatedDelta(1, 1, 1, 1, 8, 8)._ref, None) == _lib.NNSP_EINVAL
    assert L.nnsp_delta_contiguous(None) == _lib.NNSP_EINVAL
    assert L.nnsp_norm_exec_device(None, None) == _lib.NNSP_EINVAL
    assert L.nnsp_norm_contiguous(None) == _lib.NNSP_EINVAL


@pytest.mark.parametrize("sizes,message,code", [
    ((-1, 8), "rows", -1), ((1, 0), "dim", -2), ((1, 16385), "dim", -2), ((1 << 31, 8), "2\\^31", -2),
    ((1 << 30, 8, 2), "2\\^31", -2), ((1, 8, 0), "groups", -1),
])
def test_norm_sizes_refused(sizes, message, code):
    refused(lambda: BlockNorm(*sizes), message, code)


def norm(call=None, strides=None, field=None, sizes=(4, 8, 2), **kw):
    p = BlockNorm(*sizes, strides=strides, **kw)
    for k, v in (field or {}).items():
        setattr(p.args, k, v)
    ptrs = dict(x=BAD, y=BAD + 4096)
    ptrs.update(call or {})
    return lambda: p.exec_device(**ptrs)


@pytest.mark.parametrize("kw,message", [
    (dict(call={"x": None}), "x is NULL"), (dict(call={"y": None}), "both NULL"),
    (dict(act="silu"), "gate is NULL"), (dict(call={"x": BAD + 1}), "x is not aligned"),
    (dict(call={"res_in": BAD + 2}, res_dtype="f32"), "res_in is not aligned"),
    (dict(call={"w_post": BAD + 2}), "w_post is not aligned"), (dict(call={"b_pre": BAD + 1}), "b_pre is not aligned"),
    (dict(call={"y": BAD}, strides={"x": (32, 8)}), "needs its strides"),
    (dict(call={"res_in": BAD, "res_out": BAD}, strides={"res_in": (0, 8)}), "needs its strides"),
    (dict(call={"res_in": BAD + 4096}), "y must not be"), (dict(call={"res_out": BAD + 4096}), "y must not be"),
    (dict(call={"res_out": BAD}), "res_out must not be"),
    (dict(strides={"y": (8, 8)}), "coincide"), (dict(strides={"y": (0, 8)}), "coincide"),
    (dict(call={"res_out": BAD + 8192}, strides={"res_out": (12, 8)}), "coincide"),
    (dict(strides={"x": (-1, 8)}), "x stride"),
    (dict(field={"dtype": 3}), "unknown dtype"), (dict(field={"res_dtype": 2}), "res_dtype"),
    (dict(field={"post": 3}), "unknown norm"), (dict(field={"pre": -1}), "unknown norm"),
    (dict(field={"act": 9}), "unknown gate"), (dict(res_scale=float("nan")), "finite"), (dict(eps=-1e-6), "finite"),
])
def test_norm_refused(kw, message):
    refused(norm(**kw), message)


def test_norm_no_rows():
    norm(sizes=(0, 8, 2))()
