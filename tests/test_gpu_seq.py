"""Sequence operators on the GPU (include/nnsp_seq.h) against plain
implementations in 64 bits.

Tolerances, per value, relative to the scale of what is summed:
  * an output is rounded once to its type: eps / 2 of the value (finfo(t).eps / 2:
    bf16 2^-8, fp16 2^-11, fp32 2^-24);
  * before that, a delta-rule value is a sum of products each off by a few
    2^-24 (32-bit arithmetic; operands split into two 16-bit parts carry 22 bits,
    2^-23 each), over at most dk terms per frame, and the recurrence with
    |beta k k^T| <= 1 does not grow an error: n frames add theirs up.  With errors
    of random sign the sum over n frames and dk terms grows as the root, so
    2^-22 * sqrt(n * dk) * the largest magnitude bounds it with room; for 16-bit
    outputs the output's own products may use operands of 11 bits (2^-12 each,
    three of them): 3 * 2^-12 * largest / sqrt(dk) * sqrt(dk), taken as 2^-10 of
    the row's largest for bf16 only.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {t: torch.finfo(d).eps / 2 for t, d in DT.items()}


def gated_delta():
    from nnsp_amd.seq import GatedDelta
    return GatedDelta


def block_norm():
    from nnsp_amd.seq import BlockNorm
    return BlockNorm


def ptr(t):
    return None if t is None else t.data_ptr()


def delta_ref(q, k, v, g, beta, state, lens, l2norm, scale, eps=1e-6):
    """The rule, frame by frame in 64 bits, on the CPU."""
    q, k, v, beta = (x.double().cpu() for x in (q, k, v, beta))
    S, T, hv = v.shape[:3]
    g = torch.zeros(S, T, hv, dtype=torch.float64) if g is None else g.double().cpu()
    lens = [T] * S if lens is None else lens
    rep = hv // q.shape[2]
    q, k = q.repeat_interleave(rep, 2), k.repeat_interleave(rep, 2)
    if l2norm:
        q = q / (q.square().sum(-1, keepdim=True) + eps).sqrt()
        k = k / (k.square().sum(-1, keepdim=True) + eps).sqrt()
    st = torch.zeros(S, hv, q.shape[-1], v.shape[-1], dtype=torch.float64) if state is None else state.double().cpu().clone()
    out = torch.zeros(v.shape, dtype=torch.float64)
    for s in range(S):
        for t in range(lens[s]):
            new = st[s] * torch.exp(g[s, t])[:, None, None]
            u = beta[s, t][:, None] * (v[s, t] - (new * k[s, t][..., None]).sum(1))
            st[s] = new + k[s, t][..., None] * u[:, None, :]
            out[s, t] = scale * (st[s] * q[s, t][..., None]).sum(1)
    return out, st


def make(S, T, hk, hv, dk, dv, dtype, seed=0, l2norm=True, decay=1.0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k, v = rn(S, T, hk, dk), rn(S, T, hk, dk) + rn(S, 1, hk, dk), rn(S, T, hv, dv)
    if not l2norm:
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    g = -decay * torch.exp(rn(S, T, hv) - 2)
    d = {"q": q.to(DT[dtype]), "k": k.to(DT[dtype]), "v": v.to(DT[dtype]), "g": g, "beta": torch.sigmoid(rn(S, T, hv)),
         "state": 0.3 * rn(S, hv, dk, dv)}
    return {n: x.cuda() for n, x in d.items()}


def close(got, ref, dtype, T, dk, what):
    """See the module's head: one rounding to the type, plus the 32-bit sums' part."""
    got, big = got.double().cpu(), float(ref.abs().max()) if ref.numel() else 0.0
    part = 2.0 ** -22 * np.sqrt(max(1, T) * dk) + (2.0 ** -10 if dtype == "bf16" else 0.0)
    bound = HALF[dtype] * ref.abs() * (1 + part) + part * big
    off = (got - ref).abs()
    assert bool((off <= bound).all()), f"{what}: off {float((off - bound).max()):.3g} beyond the bound, largest {big:.3g}"


def run_delta(d, hk, dtype, l2norm=True, lens=None, state=True, out=None, state_out=None, stream=None, strides=None, eps=1e-6):
    S, T, hv, dv = d["v"].shape
    dk = d["q"].shape[-1]
    p = gated_delta()(S, T, hk, hv, dk, dv, dtype=dtype, l2norm=l2norm, strides=strides, eps=eps)
    out = torch.full((S, T, hv, dv), 7.0, dtype=DT[dtype], device="cuda") if out is None else out
    so = torch.full((S, hv, dk, dv), 7.0, device="cuda") if state_out is None else state_out
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(16, p.workspace_bytes), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()  # the call may go to another stream than the one that made its buffers
    p.exec_device(ptr(d["q"]), ptr(d["k"]), ptr(d["v"]), ptr(d["g"]), ptr(d["beta"]), ptr(out),
                  state_in=ptr(d["state"]) if state else None, state_out=ptr(so), lens=ptr(ln), workspace=ptr(ws),
                  stream=stream if stream is not None else torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return out, so


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("S,T,hk,hv,dk,dv", [
    (1, 1, 1, 1, 64, 64), (3, 1, 2, 4, 128, 128), (5, 2, 1, 3, 72, 40), (2, 7, 2, 2, 28, 28), (2, 5, 1, 1, 1, 1),
    (2, 4, 1, 2, 3, 5), (1, 6, 1, 1, 29, 33), (2, 3, 1, 1, 256, 256), (2, 3, 1, 1, 200, 31), (3, 8, 1, 1, 96, 65),
    (2, 9, 1, 2, 64, 64), (1, 63, 1, 1, 64, 32), (2, 64, 1, 2, 64, 64), (2, 65, 2, 2, 128, 128), (1, 130, 1, 2, 72, 96),
    (2, 100, 1, 1, 61, 47), (1, 129, 1, 1, 192, 136), (1, 70, 1, 1, 256, 256), (1, 200, 1, 1, 16, 8), (1, 66, 1, 1, 7, 3),
])
def test_delta(S, T, hk, hv, dk, dv, dtype):
    d = make(S, T, hk, hv, dk, dv, dtype, seed=S + T + dk)
    out, so = run_delta(d, hk, dtype)
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], None, True, dk ** -0.5)
    close(out, ro, dtype, T, dk, "out")
    close(so, rs, "f32", T, dk, "state")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [3, 64, 150, 300])
def test_delta_given_keys_no_decay_no_state(T, dtype):
    d = make(2, T, 1, 2, 64, 48, dtype, seed=T, l2norm=False)
    d["g"] = None
    out, so = run_delta(d, 1, dtype, l2norm=False, state=False)
    ro, rs = delta_ref(d["q"], d["k"], d["v"], None, d["beta"], None, None, False, 64 ** -0.5)
    close(out, ro, dtype, T, 64, "out")
    close(so, rs, "f32", T, 64, "state")


@pytest.mark.parametrize("T", [5, 150, 300])
def test_delta_equal_keys_and_full_beta(T):
    """The hardest triangular system: every key the same, beta 1, no decay."""
    d = make(1, T, 1, 1, 64, 64, "f32", seed=9)
    d["k"][:] = d["k"][:, :1]
    d["beta"][:] = 1.0
    d["g"][:] = 0.0
    out, so = run_delta(d, 1, "f32")
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], None, True, 64 ** -0.5)
    close(out, ro, "f32", T, 64, "out")
    close(so, rs, "f32", T, 64, "state")


@pytest.mark.parametrize("T", [4, 140, 300])
def test_delta_decays_from_nothing_to_everything(T):
    """g of 0, tiny, large and -inf: frames after a cleared state see nothing of it."""
    d = make(2, T, 1, 3, 64, 64, "bf16", seed=3)
    gen = torch.Generator().manual_seed(1)
    pick = torch.tensor([0.0, -1e-6, -0.5, -30.0, -90.0, -1000.0, float("-inf")])
    d["g"] = pick[torch.randint(0, 7, (2, T, 3), generator=gen)].cuda()
    out, so = run_delta(d, 1, "bf16")
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], None, True, 64 ** -0.5)
    close(out, ro, "bf16", T, 64, "out")
    close(so, rs, "f32", T, 64, "state")


@pytest.mark.parametrize("exponent", [-40, 40])
@pytest.mark.parametrize("T", [2, 80, 280])
def test_delta_scales(T, exponent):
    """Values far from 1 (bf16 has the range): nothing is lost to a narrower one on the way."""
    d = make(1, T, 1, 1, 64, 64, "bf16", seed=5)
    for n in ("v", "state"):
        d[n] = d[n] * 2.0 ** exponent
    d["k"] = d["k"] * 2.0 ** -exponent
    out, so = run_delta(d, 1, "bf16", l2norm=True)
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], None, True, 64 ** -0.5)
    close(out, ro, "bf16", T, 64, "out")
    close(so, rs, "f32", T, 64, "state")


@pytest.mark.parametrize("T,lens", [(6, [0, 6, 1, 5]), (100, [0, 100, 64, 65]), (200, [129, 1, 200, 63]), (70, [-3, 1000, 8, 16]), (500, [257, 1, 500, 0])])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_delta_ragged(T, lens, dtype):
    """Padding holds NaN and infinity; rows behind a stream's length keep what they held; length 0 keeps the state."""
    d = make(4, T, 1, 2, 64, 40, dtype, seed=T)
    n = [max(0, min(T, x)) for x in lens]
    for s in range(4):
        for name, junk in (("q", float("nan")), ("k", float("inf")), ("v", float("nan")), ("g", float("inf")), ("beta", float("nan"))):
            d[name][s, n[s]:] = junk
    out, so = run_delta(d, 1, dtype, lens=lens)
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], n, True, 64 ** -0.5)
    for s in range(4):
        assert bool((out[s, n[s]:] == 7).all())
        close(out[s, :n[s]], ro[s, :n[s]], dtype, T, 64, f"out {s}")
        close(so[s], rs[s], "f32", T, 64, f"state {s}")
        if n[s] == 0:
            assert torch.equal(so[s], d["state"][s])


@pytest.mark.parametrize("T", [1, 3, 66, 300])
def test_delta_strides_and_offsets(T):
    """q, k, v as slices of one projection that starts at odd addresses, heads before frames in out, repeated beta."""
    S, hk, hv, dk, dv = 3, 1, 2, 24, 20
    d = make(S, T, hk, hv, dk, dv, "bf16", seed=2)
    row = 2 * dk * hk + dv * hv + 3
    buf = torch.zeros(S * T * row + 1, dtype=torch.bfloat16, device="cuda")
    flat = buf[1:].view(S, T, row)
    flat[..., :dk] = d["q"][:, :, 0]
    flat[..., dk:2 * dk] = d["k"][:, :, 0]
    flat[..., 2 * dk:2 * dk + hv * dv] = d["v"].reshape(S, T, hv * dv)
    beta = d["beta"][:, :1, :1].contiguous()
    out = torch.full((S, hv, T, dv), 7.0, dtype=torch.bfloat16, device="cuda")
    so = torch.empty(S, hv, dk, dv, device="cuda")
    p = gated_delta()(S, T, hk, hv, dk, dv, strides={
        "q": (T * row, row, dk), "k": (T * row, row, dk), "v": (T * row, row, dv), "out": (hv * T * dv, dv, T * dv),
        "beta": (1, 0, 0)})
    ws = torch.empty(max(16, p.workspace_bytes), dtype=torch.uint8, device="cuda")
    p.exec_device(flat.data_ptr(), flat[..., dk:].data_ptr(), flat[..., 2 * dk:].data_ptr(), ptr(d["g"]), ptr(beta), ptr(out),
                  state_in=ptr(d["state"]), state_out=ptr(so), workspace=ptr(ws))
    torch.cuda.synchronize()
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], beta.expand(S, T, hv), d["state"], None, True, dk ** -0.5)
    close(out.movedim(1, 2), ro, "bf16", T, dk, "out")
    close(so, rs, "f32", T, dk, "state")


@pytest.mark.parametrize("T", [1, 90, 600])
def test_delta_state_in_place(T):
    d = make(3, T, 2, 2, 64, 64, "bf16", seed=4)
    ref_out, ref_state = run_delta(d, 2, "bf16")
    st = d["state"].clone()
    out, so = run_delta(dict(d, state=st), 2, "bf16", state_out=st)
    assert torch.equal(out, ref_out) and torch.equal(st, ref_state)


def test_delta_no_frames_copies_the_state():
    d = make(2, 0, 1, 1, 16, 16, "bf16")
    _, so = run_delta(d, 1, "bf16")
    assert torch.equal(so, d["state"])
    _, so = run_delta(d, 1, "bf16", state=False)
    assert not bool(so.any())


def test_delta_no_frames_with_lens():
    """Lengths are cut to the call's no frames; lengths in host memory are refused, not read."""
    d = make(2, 0, 1, 1, 16, 16, "bf16")
    _, so = run_delta(d, 1, "bf16", lens=[5, -1])
    assert torch.equal(so, d["state"])
    host, so = np.zeros(2, np.int32), torch.zeros_like(so)
    with pytest.raises(RuntimeError, match="lens is not memory of device"):
        gated_delta()(2, 0, 1, 1, 16, 16).exec_device(None, None, None, None, None, None, state_in=ptr(d["state"]),
                                                      state_out=ptr(so), lens=host.ctypes.data)
    torch.cuda.synchronize()
    assert not bool(so.any())


def test_delta_chunks_then_frames():
    """A stream taken in pieces of any length ends where one call ends."""
    T, cuts = 210, [0, 100, 101, 102, 166, 170, 210]
    d = make(2, T, 1, 2, 64, 64, "f32", seed=8)
    whole, final = run_delta(d, 1, "f32")
    st, parts = d["state"], []
    for a, b in zip(cuts, cuts[1:]):
        piece = {n: d[n][:, a:b].contiguous() for n in ("q", "k", "v", "g", "beta")}
        o, st = run_delta(dict(piece, state=st), 1, "f32")
        parts.append(o)
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], None, True, 64 ** -0.5)
    for o, s, what in ((whole, final, "whole"), (torch.cat(parts, 1), st, "pieces")):
        close(o, ro, "f32", T, 64, what)
        close(s, rs, "f32", T, 64, what + " state")


def delta_ref_all(d, l2norm, scale, eps=1e-6):
    """The rule in 64 bits on the GPU, all streams and heads of a frame at once."""
    q, k, v, g, beta, st = (d[n].double() for n in ("q", "k", "v", "g", "beta", "state"))
    rep = v.shape[2] // q.shape[2]
    if l2norm:
        q = q / (q.square().sum(-1, keepdim=True) + eps).sqrt()
        k = k / (k.square().sum(-1, keepdim=True) + eps).sqrt()
    out = torch.empty_like(v)
    for t in range(v.shape[1]):
        kt, qt = k[:, t].repeat_interleave(rep, 1), q[:, t].repeat_interleave(rep, 1)
        st = st * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t][..., None] * (v[:, t] - (st * kt[..., None]).sum(2))
        st = st + kt[..., None] * u[..., None, :]
        out[:, t] = scale * (st * qt[..., None]).sum(2)
    return out.cpu(), st.cpu()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("S,T,hk,hv,dk,dv", [
    (1100, 70, 1, 1, 32, 32), (600, 130, 1, 2, 64, 64), (280, 100, 2, 4, 128, 128), (520, 75, 1, 2, 61, 100),  # many streams
    (1030, 20, 1, 1, 96, 40),
    (8, 330, 32, 32, 128, 128), (9, 300, 16, 32, 104, 72),  # few, and more images than a slab holds
])
def test_delta_many_streams_and_slabs(S, T, hk, hv, dk, dv, dtype):
    d = make(S, T, hk, hv, dk, dv, dtype, seed=S)
    out, so = run_delta(d, hk, dtype)
    ro, rs = delta_ref_all(d, True, dk ** -0.5)
    close(out, ro, dtype, T, dk, "out")
    close(so, rs, "f32", T, dk, "state")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("S,T,hk,hv,dk,dv", [
    (3, 3, 1, 2, 136, 24), (2, 40, 1, 2, 256, 256), (1, 33, 2, 2, 144, 200), (2, 64, 1, 1, 129, 100), (1, 31, 1, 1, 250, 7),
    (600, 37, 1, 1, 160, 128), (1100, 66, 1, 1, 200, 64), (3, 300, 1, 2, 256, 72), (2, 560, 4, 8, 192, 144), (1, 200, 1, 3, 133, 61),
])
def test_delta_wide_keys(S, T, hk, hv, dk, dv, dtype):
    d = make(S, T, hk, hv, dk, dv, dtype, seed=S + T)
    out, so = run_delta(d, hk, dtype)
    ro, rs = delta_ref_all(d, True, dk ** -0.5)
    close(out, ro, dtype, T, dk, "out")
    close(so, rs, "f32", T, dk, "state")


@pytest.mark.parametrize("S,T,hk,hv,dk,dv,dtype", [
    (2, 1800, 32, 32, 128, 128, "bf16"), (2, 1100, 32, 32, 128, 128, "f32"), (1, 1700, 16, 32, 256, 144, "f16"),
    (12, 1300, 8, 8, 128, 104, "bf16"),
])
def test_delta_two_passes_over_several_slabs(S, T, hk, hv, dk, dv, dtype):
    d = make(S, T, hk, hv, dk, dv, dtype, seed=S)
    lens = [max(0, T - 700 * i) for i in range(S)]
    out, so = run_delta(d, hk, dtype, lens=lens)
    whole = {k: d[k] for k in d}
    for s, n in enumerate(lens):  # frames that change nothing take the place of those behind a stream's end
        whole["g"][s, n:], whole["beta"][s, n:] = 0, 0
    ro, rs = delta_ref_all(whole, True, dk ** -0.5)
    for s, n in enumerate(lens):
        assert bool((out[s, n:] == 7).all())
        close(out[s, :n], ro[s, :n], dtype, T, dk, f"out {s}")
    close(so, rs, "f32", T, dk, "state")


@pytest.mark.parametrize("state", [True, False])
def test_delta_slabs_ragged(state):
    """Streams that end in the first slab, in the middle and in the last; the final state dropped or kept."""
    S, T, h, d_ = 8, 330, 32, 128
    lens = [0, 5, 64, 190, 191, 200, 329, 330]
    d = make(S, T, h, h, d_, d_, "f32", seed=77)
    out, so = run_delta(d, h, "f32", lens=lens, state=state)
    for s, n in enumerate(lens):
        one = {k: v[s:s + 1] for k, v in d.items()}
        one = {k: (v[:, :n].contiguous() if k != "state" else v if state else torch.zeros_like(v)) for k, v in one.items()}
        ro, rs = delta_ref_all(one, True, d_ ** -0.5)
        assert bool((out[s, n:] == 7).all())
        close(out[s:s + 1, :n], ro, "f32", T, d_, f"out {s}")
        close(so[s:s + 1], rs, "f32", T, d_, f"state {s}")


@pytest.mark.parametrize("T", [5, 60, 140, 300])
def test_delta_keys_of_zeros_and_of_all_lengths(T):
    """Silence (keys and queries of zeros, also with eps 0) and frames far quieter than their neighbours."""
    for dtype in ("bf16", "f16", "f32"):
        d = make(2, T, 1, 2, 64, 64, dtype, seed=31)
        quiet = 2.0 ** -torch.arange(T, dtype=torch.float32).remainder(13).cuda()[None, :, None, None]
        d["k"], d["q"] = (d["k"].float() * quiet).to(DT[dtype]), (d["q"].float() * quiet.flip(1)).to(DT[dtype])
        d["k"][:, 1::7] = 0
        d["q"][:, 2::5] = 0
        out, so = run_delta(d, 1, dtype)
        ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], None, True, 64 ** -0.5)
        close(out, ro, dtype, T, 64, "out")
        close(so, rs, "f32", T, 64, "state")


@pytest.mark.parametrize("l2norm,qe,ke", [(True, -80, 0), (True, 0, -80), (True, 75, 75), (False, -75, 0), (False, 75, -75),
                                          (False, -75, 75)])
@pytest.mark.parametrize("T", [5, 40, 300])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_delta_rows_whose_squares_leave_32_bits(dtype, T, l2norm, qe, ke):
    """Queries and keys so faint or loud that their squares are 0 or infinite in 32 bits."""
    d = make(2, T, 1, 2, 64, 48, dtype, seed=T, l2norm=l2norm)
    d["q"], d["k"] = (d["q"].float() * 2.0 ** qe).to(DT[dtype]), (d["k"].float() * 2.0 ** ke).to(DT[dtype])
    if (l2norm, ke) == (False, 75):
        d["k"][:, 1:] = 0  # one key per stream: with more, the rule itself leaves 32 bits
    out, so = run_delta(d, 1, dtype, l2norm=l2norm, state=False)
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], None, None, l2norm, 64 ** -0.5)
    close(out, ro, dtype, T, 64, "out")
    close(so, rs, "f32", T, 64, "state")


@pytest.mark.parametrize("T", [5, 40, 150, 300])
@pytest.mark.parametrize("what", ["v", "state"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_delta_infinity_is_seen(dtype, what, T):
    """An infinite value never turns its neighbours' columns into finite wrong ones; earlier chunks are as without it."""
    d = make(2, T, 1, 2, 64, 64, dtype, seed=T)
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], None, True, 64 ** -0.5)
    t, hit = T - 3, torch.zeros(2, 2, dtype=torch.bool)
    hit[1, 1] = True
    if what == "v":
        d["v"][1, t, 1, 5] = float("inf")
    else:
        d["state"][1, 1, 7, 5], t = float("-inf"), 0
    out, so = run_delta(d, 1, dtype)
    for s, h in ((0, 0), (0, 1), (1, 0)):
        close(out[s, :, h], ro[s, :, h], dtype, T, 64, "another head")
        close(so[s, h], rs[s, h], "f32", T, 64, "another head's state")
    mine, ref = out[1, :, 1].double().cpu(), ro[1, :, 1]
    close(out[1, :t // 64 * 64, 1], ref[:t // 64 * 64], dtype, T, 64, "before")
    assert not bool(torch.isfinite(mine[t:, 5]).any()) and not bool(torch.isfinite(so[1, 1, :, 5]).any())
    fin = torch.isfinite(mine)
    close(torch.where(fin, mine, ref), ref, dtype, T, 64, "finite values")
    st = so[1, 1].double().cpu()
    close(torch.where(torch.isfinite(st), st, rs[1, 1]), rs[1, 1], "f32", T, 64, "finite states")


@pytest.mark.parametrize("S,T,h,d_", [(2, 5, 2, 64), (2, 130, 2, 64), (2, 500, 2, 64), (2, 1800, 32, 128), (300, 70, 1, 32)])
def test_delta_final_state_dropped(S, T, h, d_):
    """Frame by frame, in chunks (few rows and many) and in two passes (of one slab and of several), without state_out."""
    d = make(S, T, h, h, d_, d_, "bf16", seed=S)
    ref, _ = run_delta(d, h, "bf16")
    p = gated_delta()(S, T, h, h, d_, d_)
    out = torch.zeros_like(ref)
    ws = torch.empty(max(16, p.workspace_bytes), dtype=torch.uint8, device="cuda")
    p.exec_device(ptr(d["q"]), ptr(d["k"]), ptr(d["v"]), ptr(d["g"]), ptr(d["beta"]), ptr(out), state_in=ptr(d["state"]),
                  workspace=ptr(ws), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(out, ref)


def test_delta_two_calls_at_once():
    """Two calls in two passes on two streams, each with its own workspace, and one more behind the first."""
    T = 700
    d = [make(2, T, 2, 4, 128, 128, "bf16", seed=i) for i in range(2)]
    ref = [run_delta(x, 2, "bf16") for x in d]
    p = gated_delta()(2, T, 2, 4, 128, 128)
    st = [torch.cuda.Stream() for _ in d]
    ws = [torch.empty(p.workspace_bytes, dtype=torch.uint8, device="cuda") for _ in d]
    out, so = [torch.zeros_like(r[0]) for r in ref], [torch.zeros_like(r[1]) for r in ref]
    torch.cuda.synchronize()
    for i in (0, 1, 0):
        p.exec_device(ptr(d[i]["q"]), ptr(d[i]["k"]), ptr(d[i]["v"]), ptr(d[i]["g"]), ptr(d[i]["beta"]), ptr(out[i]),
                      state_in=ptr(d[i]["state"]), state_out=ptr(so[i]), workspace=ptr(ws[i]), stream=st[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(out[i], ref[i][0]) and torch.equal(so[i], ref[i][1])


@pytest.mark.parametrize("T", [1, 7, 40, 300])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_delta_rows_of_zeros_without_eps(dtype, T):
    """Nothing is divided by the length of a row that has none."""
    d = make(2, T, 1, 2, 64, 40, dtype, seed=T)
    d["k"][0, ::3], d["q"][1, ::2] = 0, 0
    d["k"][1, -1:], d["q"][0, -1:] = 0, 0
    out, so = run_delta(d, 1, dtype, eps=0.0)
    # the oracle's 1e-60 changes no other length
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], None, True, 64 ** -0.5, eps=1e-60)
    close(out, ro, dtype, T, 64, "out")
    close(so, rs, "f32", T, 64, "state")


@pytest.mark.parametrize("T", [6, 40, 150, 300])
def test_delta_growth(T):
    """Decays above 1 now and then, as a learned gate may give: what a state gains over 64 frames stays small."""
    d = make(2, T, 1, 2, 64, 40, "f32", seed=T)
    d["g"] = 0.05 * torch.randn(2, T, 2, generator=torch.Generator().manual_seed(T)).cuda()
    out, so = run_delta(d, 1, "f32")
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], None, True, 64 ** -0.5)
    # the largest product of decays over 64 frames is the factor that precision may cost
    s = torch.cumsum(d["g"].double().cpu(), 1)
    s = torch.cat([torch.zeros(2, 1, 2, dtype=torch.float64), s], 1)
    grow = max(float((s[:, i + 1:i + 65] - s[:, i:i + 1]).max()) for i in range(T))
    close(out, ro, "f32", T * np.exp(2 * grow), 64, "out")
    close(so, rs, "f32", T * np.exp(2 * grow), 64, "state")


def test_delta_same_bits_every_time_and_by_stream():
    """Results do not depend on the run, nor on the other streams of the call."""
    d = make(40, 130, 2, 4, 64, 64, "bf16", seed=6)
    a, sa = run_delta(d, 2, "bf16")
    b, sb = run_delta(d, 2, "bf16")
    assert torch.equal(a, b) and torch.equal(sa, sb)


@pytest.mark.parametrize("T", [1, 130, 600])
def test_delta_other_stream(T):
    d = make(2, T, 1, 2, 64, 64, "bf16", seed=7)
    ref, rs = run_delta(d, 1, "bf16")
    st = torch.cuda.Stream()
    out, so = run_delta(d, 1, "bf16", stream=st.cuda_stream)
    assert torch.equal(out, ref) and torch.equal(so, rs)


@pytest.mark.parametrize("T", [1, 130, 600])
def test_delta_in_a_graph(T):
    """Captured once, replayed on new inputs, with the same call made eagerly in between."""
    S, hk, hv, dk, dv = 2, 1, 2, 64, 64
    p = gated_delta()(S, T, hk, hv, dk, dv, dtype="bf16")
    d = make(S, T, hk, hv, dk, dv, "bf16", seed=10)
    out, so = torch.zeros_like(d["v"]), torch.zeros_like(d["state"])
    ws = torch.empty(max(16, p.workspace_bytes), dtype=torch.uint8, device="cuda")

    def call():
        p.exec_device(ptr(d["q"]), ptr(d["k"]), ptr(d["v"]), ptr(d["g"]), ptr(d["beta"]), ptr(out), state_in=ptr(d["state"]),
                      state_out=ptr(so), workspace=ptr(ws), stream=torch.cuda.current_stream().cuda_stream)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in (11, 12, 13):
        for n, x in make(S, T, hk, hv, dk, dv, "bf16", seed=seed).items():
            d[n].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got, gs = out.clone(), so.clone()
        out.zero_(), so.zero_()
        call()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(gs, so)


@pytest.mark.parametrize("T", [3, 40, 300])
def test_delta_far_offsets(T):
    """Streams more than 2^31 elements apart, one frame at a time, in chunks and in two passes."""
    dk, dv, far = 16, 16, 1 << 31
    d = make(2, T, 1, 1, dk, dv, "bf16", seed=14)
    buf = torch.zeros(far + T * dv, dtype=torch.bfloat16, device="cuda")
    v = torch.as_strided(buf, (2, T, 1, dv), (far, dv, dv, 1), 0)
    v.copy_(d["v"])
    out, so = torch.zeros(2, T, 1, dv, dtype=torch.bfloat16, device="cuda"), torch.zeros_like(d["state"])
    p = gated_delta()(2, T, 1, 1, dk, dv, strides={"v": (far, dv, dv)})
    ws = torch.empty(max(16, p.workspace_bytes), dtype=torch.uint8, device="cuda")
    p.exec_device(ptr(d["q"]), ptr(d["k"]), buf.data_ptr(), ptr(d["g"]), ptr(d["beta"]), ptr(out), state_in=ptr(d["state"]),
                  state_out=ptr(so), workspace=ptr(ws))
    torch.cuda.synchronize()
    ro, rs = delta_ref(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], None, True, dk ** -0.5)
    close(out, ro, "bf16", T, dk, "out")
    close(so, rs, "f32", T, dk, "state")


@pytest.mark.parametrize("T", [2, 50])
def test_delta_pinned_host_memory(T):
    """Inputs and the state in pinned host memory, which the device reads and writes in place."""
    d = make(2, T, 1, 2, 64, 40, "bf16", seed=T)
    ref, rs = run_delta(d, 1, "bf16")
    pinned = {n: torch.empty(x.shape, dtype=x.dtype, pin_memory=True).copy_(x) for n, x in d.items()}
    so = torch.zeros(rs.shape, pin_memory=True)
    out, _ = run_delta(pinned, 1, "bf16", state_out=so)
    assert torch.equal(out, ref) and torch.equal(so, rs.cpu())


def test_delta_host_memory_is_refused():
    d = make(1, 1, 1, 1, 16, 16, "bf16")
    p = gated_delta()(1, 1, 1, 1, 16, 16)
    host = np.zeros(64, np.float32)
    with pytest.raises(RuntimeError, match="is not memory of device"):
        p.exec_device(ptr(d["q"]), ptr(d["k"]), ptr(d["v"]), ptr(d["g"]), host.ctypes.data, ptr(d["v"]) + 1024)
    torch.cuda.synchronize()  # nothing was queued, no error is left behind
    out, _ = run_delta(d, 1, "bf16")
    assert bool(torch.isfinite(out).all())


# ---- norms -------------------------------------------------------------------

def norm_ref(x, gate, res, w, dim, post, act, pre, scale, col, eps=1e-6):
    def norm(x, kind, wt, b):
        if kind == "none":
            return x
        if kind == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        x = x if wt is None else x * wt.double().cpu()
        return x if b is None else x + b.double().cpu()

    h = norm(x.double().cpu(), post, w.get("w_post"), w.get("b_post"))
    if act != "none":
        z = gate.double().cpu()
        h = h * torch.sigmoid(z) * (z if act == "silu" else 1)
    r = scale * h * (1 if col is None else col.double().cpu())
    r = r if res is None else r + res.double().cpu()
    return norm(r, pre, w.get("w_pre"), w.get("b_pre")), r


def norm_close(got, ref, dtype, dim, what):
    """One rounding to the type; sums of dim terms in 32 bits (tree sums: 2^-24 sqrt(dim) of the row's scale) and about
    16 operations of 2^-23 each between (exp and reciprocals are good to one unit)."""
    got, ref = got.double().cpu(), ref
    big = ref.abs().amax(-1, keepdim=True)
    part = 2.0 ** -24 * np.sqrt(dim) + 16 * 2.0 ** -23
    bound = HALF[dtype] * ref.abs() * (1 + part) + part * big + torch.finfo(DT[dtype]).tiny
    off = (got - ref).abs()
    assert bool((off <= bound).all()), f"{what}: {float((off - bound).max()):.3g} beyond the bound"


def norm_inputs(rows, groups, dim, dtype, res, seed):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, gate, r = (rn(rows, groups, dim).to(DT[dtype]).cuda() for _ in range(3))
    r = None if res is None else (2 * rn(rows, groups, dim)).to(DT[res]).cuda()
    w = {n: ((1 if n[0] == "w" else 0) + 0.2 * rn(dim)).cuda() for n in ("w_post", "b_post", "w_pre", "b_pre")}
    return x, gate, r, w, rn(dim).cuda()


@pytest.mark.parametrize("dtype,res", [("bf16", None), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("rows,groups,dim", [(1, 1, 1), (3, 2, 7), (5, 1, 64), (33, 3, 65), (2, 1, 129), (9, 1, 256), (3, 1, 1000),
                                             (2, 2, 1025), (5, 1, 1383), (7, 1, 1536), (2, 1, 1537), (2, 1, 2048), (3, 1, 4097), (1, 1, 8192), (2, 1, 16384), (1, 1, 16383)])
@pytest.mark.parametrize("post,act,pre", [("rms", "sigmoid", "rms"), ("layer", "silu", "layer"), ("none", "none", "rms"),
                                          ("rms", "silu", "none")])
def test_norm(rows, groups, dim, dtype, res, post, act, pre):
    x, gate, r, w, col = norm_inputs(rows, groups, dim, dtype, res, dim + rows)
    full = pre == "layer"
    y = torch.zeros_like(x)
    ro = None if r is None else torch.zeros_like(r)
    p = block_norm()(rows, dim, groups, dtype=dtype, res_dtype=res, post=post, act=act, pre=pre, res_scale=0.7)
    use = {n: t for n, t in w.items() if full or n[0] == "w"}
    p.exec_device(ptr(x), ptr(y), gate=ptr(gate) if act != "none" else None, col_scale=ptr(col) if full else None,
                  res_in=ptr(r), res_out=ptr(ro), **{n: ptr(t) for n, t in use.items()})
    torch.cuda.synchronize()
    ref_y, ref_r = norm_ref(x, gate, r, use, dim, post, act, pre, 0.7, col if full else None)
    norm_close(y, ref_y, dtype, dim, "y")
    if r is not None:
        norm_close(ro, ref_r, res, dim, "res_out")


def test_norm_layer_of_one_value():
    x, gate, r, w, _ = norm_inputs(3, 1, 1, "f32", "f32", 1)
    y, ro = torch.zeros_like(x), torch.zeros_like(x)
    block_norm()(3, 1, dtype="f32", post="layer", pre="layer").exec_device(
        ptr(x), ptr(y), res_in=ptr(r), res_out=ptr(ro), **{n: ptr(t) for n, t in w.items()})
    torch.cuda.synchronize()
    assert torch.equal(y[:, 0, 0], w["b_pre"].expand(3)) and torch.equal(ro, r + w["b_post"])


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norm_zero_constant_and_offset_rows(kind):
    """A row of zeros, one of a constant, one with a mean far above its spread."""
    dim = 512
    x = torch.zeros(3, 1, dim, device="cuda")
    x[1] = 3.0
    x[2] = 1000.0 + torch.randn(dim, generator=torch.Generator().manual_seed(0)).cuda()
    y = torch.full_like(x, 7.0)
    block_norm()(3, dim, dtype="f32", post="none", pre=kind).exec_device(ptr(x), ptr(y))
    torch.cuda.synchronize()
    ref, _ = norm_ref(x, None, None, {}, dim, "none", "none", kind, 1.0, None)
    # the mean of the third row is 1000 and rounded to 2^-24 of that: what is left of it shows in the layer norm
    extra = 1000 * 2.0 ** -23 if kind == "layer" else 0.0
    off = (y.double().cpu() - ref).abs()
    assert bool((off <= 2.0 ** -18 * ref.abs().amax(-1, keepdim=True) + extra).all())
    assert not bool(y[0].any())


def test_norm_strides_in_place_and_what_is_not_written():
    rows, groups, dim = 6, 3, 50
    x, gate, r, w, _ = norm_inputs(rows, groups, dim, "bf16", "bf16", 3)
    wide = torch.full((rows, groups, dim + 5), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[..., :dim] = x
    st = (groups * (dim + 5), dim + 5)
    one_gate = gate[:, :1].contiguous()  # one gate for all heads
    res = r.clone()
    p = block_norm()(rows, dim, groups, act="silu", strides={"x": st, "y": st, "gate": (dim, 0)})
    p.exec_device(ptr(wide), ptr(wide), gate=ptr(one_gate), res_in=ptr(res), res_out=ptr(res), w_pre=ptr(w["w_pre"]))
    torch.cuda.synchronize()
    ref_y, ref_r = norm_ref(x, one_gate.expand(rows, groups, dim), r, {"w_pre": w["w_pre"]}, dim, "rms", "silu", "rms", 1.0, None)
    norm_close(wide[..., :dim], ref_y, "bf16", dim, "y")
    norm_close(res, ref_r, "bf16", dim, "res_out")
    assert bool((wide[..., dim:] == 7).all())
    only = torch.zeros_like(r)
    block_norm()(rows, dim, groups, pre="rms").exec_device(ptr(x), None, res_in=ptr(r), res_out=ptr(only))
    torch.cuda.synchronize()
    norm_close(only, norm_ref(x, None, r, {}, dim, "rms", "none", "rms", 1.0, None)[1], "bf16", dim, "res_out alone")


def test_norm_rows_do_not_mix():
    """A row of NaN leaves its neighbours alone (rows share a wave here)."""
    x = torch.randn(40, 1, 64, generator=torch.Generator().manual_seed(2)).cuda()
    y = torch.zeros_like(x)
    block_norm()(40, 64, dtype="f32").exec_device(ptr(x), ptr(y))
    x[7] = float("nan")
    x[9, 0, 3] = float("inf")
    z = torch.zeros_like(x)
    block_norm()(40, 64, dtype="f32").exec_device(ptr(x), ptr(z))
    torch.cuda.synchronize()
    keep = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(y[keep], z[keep]) and bool(torch.isnan(z[7]).all())


def test_norm_in_a_graph():
    x, gate, r, w, _ = norm_inputs(20, 1, 2048, "bf16", "f32", 5)
    y, ro = torch.zeros_like(x), torch.zeros_like(r)
    p = block_norm()(20, 2048, res_dtype="f32", act="silu")

    def call():
        p.exec_device(ptr(x), ptr(y), gate=ptr(gate), w_pre=ptr(w["w_pre"]), res_in=ptr(r), res_out=ptr(ro),
                      stream=torch.cuda.current_stream().cuda_stream)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in range(3):
        x.copy_(norm_inputs(20, 1, 2048, "bf16", "f32", 50 + seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        got, gr = y.clone(), ro.clone()
        y.zero_(), ro.zero_()
        call()
        torch.cuda.synchronize()
        assert torch.equal(got, y) and torch.equal(gr, ro)


def test_norm_more_rows_than_a_grid_has_threads_along_x():
    """2^29 + 33 rows by 8 lanes each."""
    rows = (1 << 29) + 33
    x = torch.arange(rows, device="cuda", dtype=torch.int32).remainder_(251).to(torch.bfloat16)
    y = torch.zeros_like(x)
    block_norm()(rows, 1, post="none", pre="none", res_scale=2.0).exec_device(ptr(x), ptr(y))
    torch.cuda.synchronize()
    assert torch.equal(y, x.mul_(2))


# ---- together ----------------------------------------------------------------

def test_a_layer_by_chunk_and_by_frame():
    """Delta rule, gated head norm, projection, residual norm: 2 layers over a chunk, then frame by frame from the state
    that the chunk left, against the same net in 64 bits."""
    S, T0, T1, H, d, D = 3, 70, 4, 2, 32, 64
    gen = torch.Generator().manual_seed(21)
    rn = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    layers = [{"in": rn(D, 4 * H * d + 2 * H) / 8, "out": rn(H * d, D) / 8, "w_post": 1 + 0.1 * rn(d), "w_pre": 1 + 0.1 * rn(D)}
              for _ in range(2)]
    x0 = rn(S, T0 + T1, D)

    def run(x, states):
        T = x.shape[1]
        res, y = x.contiguous(), torch.empty_like(x)
        block_norm()(S * T, D, dtype="f32", post="none").exec_device(ptr(res), ptr(y))
        for n, L in enumerate(layers):
            proj = (y @ L["in"]).contiguous()
            row, hd = proj.shape[-1], H * d
            g, beta = -torch.nn.functional.softplus(proj[..., 4 * hd:4 * hd + H]), torch.sigmoid(proj[..., 4 * hd + H:])
            g, beta = g.contiguous(), beta.contiguous()
            st = (T * row, row, d)
            p = gated_delta()(S, T, H, H, d, d, dtype="f32", strides={"q": st, "k": st, "v": st})
            ws = torch.empty(max(16, p.workspace_bytes), dtype=torch.uint8, device="cuda")
            o = torch.empty(S, T, H, d, device="cuda")
            p.exec_device(ptr(proj), proj[..., hd:].data_ptr(), proj[..., 2 * hd:].data_ptr(), ptr(g), ptr(beta), ptr(o),
                          state_in=ptr(states[n]), state_out=ptr(states[n]), workspace=ptr(ws))
            block_norm()(S * T, d, H, dtype="f32", post="rms", act="silu", pre="none", strides={"gate": (row, d)}).exec_device(
                ptr(o), ptr(o), gate=proj[..., 3 * hd:].data_ptr(), w_post=ptr(L["w_post"]))
            blk = (o.reshape(S, T, hd) @ L["out"]).contiguous()
            y = torch.empty_like(blk)
            block_norm()(S * T, D, dtype="f32", post="rms", pre="rms", res_scale=0.5).exec_device(
                ptr(blk), ptr(y), w_pre=ptr(L["w_pre"]), res_in=ptr(res), res_out=ptr(res))
            torch.cuda.synchronize()
        return y

    def ref():
        rms = lambda x: x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
        res = x0.double().cpu()
        y, T = rms(res), T0 + T1
        for L in layers:
            W = {n: t.double().cpu() for n, t in L.items()}
            proj = y @ W["in"]
            q, k, v, z = (proj[..., i * H * d:(i + 1) * H * d].reshape(S, T, H, d) for i in range(4))
            g, beta = -torch.nn.functional.softplus(proj[..., 4 * H * d:4 * H * d + H]), torch.sigmoid(proj[..., 4 * H * d + H:])
            o, _ = delta_ref(q, k, v, g, beta, None, None, True, d ** -0.5)
            o = rms(o) * W["w_post"] * z * torch.sigmoid(z)
            res = res + 0.5 * rms(o.reshape(S, T, H * d) @ W["out"])
            y = rms(res) * W["w_pre"]
        return y

    states = [torch.zeros(S, H, d, d, device="cuda") for _ in layers]
    got = [run(x0[:, :T0], states)] + [run(x0[:, t:t + 1], states) for t in range(T0, T0 + T1)]
    got, want = torch.cat(got, 1).double().cpu(), ref()
    # each layer ends in norms, so what one leaves off (about 2^-22 sqrt(T d) of the values) is passed on at its own
    # size; the norm of a head's output can raise a small one by the ratio of its row to the largest, 2^4 here
    assert float((got - want).abs().max()) <= 2 * 16 * 2.0 ** -22 * np.sqrt(74 * 32) * float(want.abs().max())
