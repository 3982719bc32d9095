"""Fused norms on the GPU: rows at the ends of 32 bits, long rows in place."""
import numpy as np
import pytest
import torch

from test_gpu_seq import DT, block_norm, norm_close, norm_inputs, norm_ref, ptr

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [7, 64, 100, 1024, 1383, 2048, 5000, 16384])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("exponent,eps", [(70, 1e-6), (100, 1e-6), (-70, 0.0), (-100, 0.0), (-70, 1e-41)])
def test_norm_rows_whose_squares_leave_32_bits(exponent, eps, kind, dim, dtype):
    """A row so loud or faint that its squares are infinite or 0 in 32 bits has a length all the same, before and after
    the block, beside rows of usual size."""
    gen = torch.Generator().manual_seed(dim)
    x = torch.randn(6, 1, dim, generator=gen)
    x[1::2] *= 2.0 ** exponent
    x = x.to(DT[dtype]).cuda()
    w = {n: (1 + 0.2 * torch.randn(dim, generator=gen)).cuda() for n in ("w_post", "w_pre")}
    for post, pre in ((kind, "none"), ("none", kind)):
        y = torch.zeros_like(x)
        use = {"w_post" if post != "none" else "w_pre": w["w_post" if post != "none" else "w_pre"]}
        block_norm()(6, dim, dtype=dtype, post=post, pre=pre, eps=eps).exec_device(ptr(x), ptr(y), **{n: ptr(t) for n, t in use.items()})
        torch.cuda.synchronize()
        ref, _ = norm_ref(x, None, None, use, dim, post, "none", pre, 1.0, None, eps=float(np.float32(eps)))
        norm_close(y, ref, dtype, dim, f"{post} {pre}")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [7, 50, 1383, 1537, 2049, 4100, 9001, 16383])
@pytest.mark.parametrize("post", ["none", "rms"])
def test_norm_in_place(dim, dtype, post):
    """y in place of x and of the gate, res_out in place of res_in, rows that end within a thread's elements."""
    rows = 9
    x, gate, r, w, col = norm_inputs(rows, 1, dim, dtype, dtype, dim)
    p = block_norm()(rows, dim, dtype=dtype, post=post, act="silu", pre="rms", res_scale=0.5)
    ref = [torch.zeros_like(x), torch.zeros_like(r)]
    p.exec_device(ptr(x), ptr(ref[0]), gate=ptr(gate), res_in=ptr(r), res_out=ptr(ref[1]), col_scale=ptr(col), w_pre=ptr(w["w_pre"]))
    torch.cuda.synchronize()
    norm_close(ref[0], norm_ref(x, gate, r, {"w_pre": w["w_pre"]}, dim, post, "silu", "rms", 0.5, col)[0], dtype, dim, "y")
    for at in ("x", "gate"):
        t, res = {"x": x.clone(), "gate": gate.clone()}, r.clone()
        p.exec_device(ptr(t["x"]), ptr(t[at]), gate=ptr(t["gate"]), res_in=ptr(res), res_out=ptr(res), col_scale=ptr(col),
                      w_pre=ptr(w["w_pre"]))
        torch.cuda.synchronize()
        assert torch.equal(t[at], ref[0]) and torch.equal(res, ref[1])
    # nothing between the loads and the stores but the multiplication
    y = x.clone()
    block_norm()(rows, dim, dtype=dtype, post="none", pre="none", res_scale=2.0).exec_device(ptr(y), ptr(y))
    torch.cuda.synchronize()
    assert torch.equal(y, x * 2)
