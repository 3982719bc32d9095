"""Delta rule on the GPU: every stream, head and column of the state by itself,
against the rule in 64 bits.

A column of the state, with its column of v and out, is a recurrence of its
own: S'^T k, u, S and the output's column take nothing from the columns beside
it.  So each is bounded by its own size, with big = the largest length of the
state's column over the frames (its start too) plus the largest |v| of it:

  * Within a chunk seven roundings of an operand or a sum stand between S0 and
    S1 (q or k and S0 in K S0; R, T in T R; U fk and K in K^T U; each an fp16
    pair of 22 bits, off by 2^-23 of its value, lo * lo of two pairs left out,
    2^-24; and sums in 32 bits, 2^-24 a step of a few).  By Cauchy-Schwarz each
    is off by its part of |k| |S|, whatever dk is, so all of them by less than
    8 * 2^-23 of big, and by twice that where the inverse's rows add up what
    cancels.  |beta k k^T| <= 1 lets no error grow, and errors of the frames
    have random signs: part = 16 * 2^-23 * sqrt(frames).
  * out = scale q . S: scale * part * big, and one rounding to its type (half a
    step of the value, or of the smallest subnormal).
"""
import numpy as np
import pytest
import torch

from test_gpu_seq import DT, HALF, make, run_delta

pytestmark = pytest.mark.gpu


def rule(d, scale, eps=1e-6):
    """out, the final state, and big [S][hv][dv], in 64 bits on the GPU."""
    unit = {n: d[n].double() / (d[n].double().square().sum(-1, keepdim=True) + eps).sqrt() for n in ("q", "k")}
    return rule_given(dict(d, **unit), scale)


def rule_given(d, scale):
    """The same with q and k as they are."""
    q, k, v, g, beta, st = (d[n].double() for n in ("q", "k", "v", "g", "beta", "state"))
    T, hv = v.shape[1:3]
    rep = hv // q.shape[2]
    out, big = torch.zeros_like(v), st.square().sum(2)
    for t in range(T):
        kt, qt = k[:, t].repeat_interleave(rep, 1), q[:, t].repeat_interleave(rep, 1)
        new = st * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t][..., None] * (v[:, t] - (new * kt[..., None]).sum(2))
        new = new + kt[..., None] * u[..., None, :]
        st = new
        out[:, t] = scale * (st * qt[..., None]).sum(2)
        big = torch.maximum(big, st.square().sum(2))
    return out, st, big.sqrt() + v.abs().amax(1)


def check(got, ref, scale, dtype, T):
    (out, so), (ro, rs, big) = got, ref
    part = 16 * 2.0 ** -23 * np.sqrt(T)
    least = 2.0 ** -25 if dtype == "f16" else 2.0 ** -134 if dtype == "bf16" else 2.0 ** -150
    bound = HALF[dtype] * ro.abs() + least + (scale * big * part)[:, None]
    for what, off, most in (("out", (out.double() - ro).abs(), bound), ("state", (so.double() - rs).abs(), (part * big)[:, :, None])):
        at = torch.nonzero(~(off <= most))
        assert len(at) == 0, f"{what}: {len(at)} of {off.numel()} beyond the bound, at {at[0].tolist()} by {float((off / most).max()):.3g}"


# one for each way that a call runs: frame by frame, three chunks at once, many rows (by 64 and 128 columns a workgroup, with
# waves to spare and without), wide keys, two passes by 16 and by 32 columns, and by several slabs
WAYS = [(2, 2, 1, 2, 64, 72), (2, 100, 1, 2, 64, 72), (1, 40, 2, 2, 128, 128), (2, 70, 1, 2, 61, 47), (300, 40, 1, 2, 64, 48),
        (200, 70, 1, 2, 64, 128), (140, 40, 1, 2, 128, 136), (260, 33, 1, 1, 96, 24), (3, 45, 1, 2, 200, 72), (200, 40, 1, 2, 160, 128),
        (1, 300, 1, 2, 64, 64), (2, 333, 1, 2, 128, 40), (10, 420, 2, 4, 64, 128), (9, 420, 2, 4, 128, 128), (1, 200, 1, 2, 192, 64),
        (1, 420, 1, 2, 61, 47), (1, 1900, 32, 32, 128, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("S,T,hk,hv,dk,dv", WAYS)
def test_delta_every_column_by_its_own_size(S, T, hk, hv, dk, dv, dtype):
    """Columns of all sizes side by side, fast and slow heads, loud and quiet streams."""
    d = make(S, T, hk, hv, dk, dv, dtype, seed=S + T + dv)
    low = [0, -5, -20, 3, -12] if dtype == "f16" else [0, -12, -24, 3, -40]
    col = 2.0 ** torch.tensor([low[(i * 3 + i // 16) % 5] for i in range(dv)], dtype=torch.float32).cuda()
    # fp16's own range is not as wide: nothing is written to the faintest columns there
    d["v"] = (d["v"].float() * (col * (col > 2.0 ** -10) if dtype == "f16" else col)).to(DT[dtype])
    d["state"] = d["state"] * col
    d["g"] = d["g"] * torch.tensor([4.0 ** -(h % 4) for h in range(hv)]).cuda()
    got = run_delta(d, hk, dtype)
    check(got, rule(d, dk ** -0.5), dk ** -0.5, dtype, T)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("S,T,hk,hv,dk,dv", [w for w in WAYS if w[1] < 1000])
def test_delta_columns_do_not_touch_each_other(S, T, hk, hv, dk, dv, dtype):
    """What stands in one column, be it an infinity or a NaN, changes no bit of the others."""
    d = make(S, T, hk, hv, dk, dv, dtype, seed=S + T)
    out, so = run_delta(d, hk, dtype)
    hit = [2, 17, 18, dv - 1]
    keep = [c for c in range(dv) if c not in hit]
    d["state"][:, :, 3, 2] = float("inf")
    d["v"][:, T // 2:, :, 17] = float("-inf")
    d["v"][:, T - 1, :, 18] = float("nan")
    d["v"][..., dv - 1] *= 1024
    out2, so2 = run_delta(d, hk, dtype)
    assert torch.equal(out[..., keep], out2[..., keep]) and torch.equal(so[..., keep], so2[..., keep])
    for c in (2, 17, 18):
        assert not bool(torch.isfinite(out2[:, T - 1, :, c]).any())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,T,hk,hv,dk,dv", WAYS[:-1])
def test_delta_a_stream_by_itself_and_among_others(S, T, hk, hv, dk, dv, dtype):
    """A stream's results do not depend on what the call's other streams hold (how many they are may choose another
    kernel, whose results are as exact)."""
    d = make(S, T, hk, hv, dk, dv, dtype, seed=S + dk)
    d["g"] = d["g"] * torch.tensor([4.0 ** -(h % 4) for h in range(hv)]).cuda()
    out, so = run_delta(d, hk, dtype)
    one = {n: x[-1:].contiguous() for n, x in d.items()}
    ref = rule(one, dk ** -0.5)
    check((out[-1:], so[-1:]), ref, dk ** -0.5, dtype, T)
    check(run_delta(one, hk, dtype), ref, dk ** -0.5, dtype, T)
    if S > 1:
        for x in d.values():
            x[:-1] = x[:-1].flip(0) * 3
        d["v"][0], d["k"][0] = float("nan"), float("inf")
        out2, so2 = run_delta(d, hk, dtype)
        assert torch.equal(out[-1], out2[-1]) and torch.equal(so[-1], so2[-1])


@pytest.mark.parametrize("what", ["beta", "g", "k", "q", "nan beta", "nan g", "nan k"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("S,T,t", [(1, 60, 25), (1, 60, 45), (1, 300, 168), (1, 300, 250), (300, 60, 45), (6, 420, 240)])
def test_delta_what_is_not_finite_leaves_no_wrong_frame(S, T, t, dtype, what):
    """Frames before it come out right or, in its chunk, not finite; never finite and wrong.  Keys as given."""
    hk, hv, dk, dv = 1, 2, 64, 72 if S < 6 else 128
    d = make(S, T, hk, hv, dk, dv, dtype, seed=T + t, l2norm=False)
    ro, rs, big = rule_given(d, dk ** -0.5)
    x = float("nan") if what.startswith("nan") else float("inf")
    name = what.split()[-1]
    if name in ("k", "q"):
        d[name][-1, t, 0, 3] = x
    else:
        d[name][-1, t, 1] = x
    out, so = run_delta(d, hk, dtype, l2norm=False)
    part = 16 * 2.0 ** -23 * np.sqrt(T)
    bound = HALF[dtype] * ro.abs() + (dk ** -0.5 * big * part)[:, None] + 2.0 ** -25
    fine = (out.double() - ro).abs() <= bound
    heads = [0, 1] if name in ("k", "q") else [1]
    start = t // 64 * 64 if name != "q" else t
    assert bool(fine[:-1].all()) and bool(fine[-1, :start].all()) and bool(fine[-1, :, [h for h in (0, 1) if h not in heads]].all())
    assert bool((fine | ~torch.isfinite(out))[-1, :t].all())
    if name == "q":  # only its own frame takes it
        assert bool(fine[-1, t + 1:].all()) and bool(((so.double() - rs).abs() <= (part * big)[:, :, None]).all())
        assert not bool(torch.isfinite(out[-1, t]).any())
    else:
        assert not bool(torch.isfinite(out[-1, t:, heads]).any()) and not bool(torch.isfinite(so[-1, heads]).any())


@pytest.mark.parametrize("T", [3, 40, 300])
@pytest.mark.parametrize("exponent", [-14, -17, -20])
def test_delta_faintest_keys_of_fp16(T, exponent):
    """Rows of fp16's subnormal numbers have their length too, beside eps (1e-6 is above it from 2^-14 on) and without."""
    for eps in (1e-6, 0.0):
        d = make(2, T, 1, 2, 64, 48, "f16", seed=T)
        d["q"], d["k"] = (d["q"].float() * 2.0 ** exponent).half(), (d["k"].float() * 2.0 ** exponent).half()
        got = run_delta(d, 1, "f16", eps=eps)
        check(got, rule(d, 64 ** -0.5, eps=eps or 1e-60), 64 ** -0.5, "f16", T)


@pytest.mark.parametrize("T", [1, 12])
@pytest.mark.parametrize("dk,dv,streams", [(1, 1, (1 << 24) - 1), (33, 80, ((1 << 24) - 1) // 5)])
def test_delta_as_many_streams_as_there_may_be(dk, dv, streams, T):
    """The largest grids, frame by frame and in chunks, on inputs that all streams share; the first, the last and some
    between against the rule."""
    if T > 1 and dk > 1:
        streams //= 8  # its states alone would be 35 GB
    d = make(1, T, 1, 1, dk, dv, "f32", seed=dk)
    from nnsp_amd.seq import GatedDelta
    zero = {n: (0, h * w, w) for n, h, w in (("q", 1, dk), ("k", 1, dk), ("g", 1, 1), ("beta", 1, 1))}
    p = GatedDelta(streams, T, 1, 1, dk, dv, dtype="f32", strides=dict(zero, v=(1, dv, dv)))
    v = torch.randn(streams + T * dv, generator=torch.Generator().manual_seed(1)).cuda()  # stream s: from element s on
    out = torch.full((streams, T, dv), 7.0, device="cuda")
    so = torch.full((streams, dk, dv), 7.0, device="cuda")
    assert p.workspace_bytes == 0
    p.exec_device(d["q"].data_ptr(), d["k"].data_ptr(), v.data_ptr(), d["g"].data_ptr(), d["beta"].data_ptr(), out.data_ptr(),
                  state_out=so.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    at = [0, 1, streams // 3, streams // 2 + 1, streams - 2, streams - 1]
    some = {n: d[n].expand(len(at), *d[n].shape[1:]) for n in ("q", "k", "g", "beta")}
    some["v"] = torch.stack([v[s:s + T * dv].view(T, 1, dv) for s in at])
    some["state"] = torch.zeros(len(at), 1, dk, dv, device="cuda")
    check((out[at][:, :, None], so[at][:, None]), rule(some, dk ** -0.5), dk ** -0.5, "f32", T)
    assert bool((so != 7).any(-1).any(-1).all())
