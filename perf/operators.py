"""What the sequence-layer operators are measured on: the gated delta rule (a
chunk of frames, one frame) and the norms around a block, fused with its gate
and residual scale.  Plain forms in elementary torch operations, 32 bits (64
where 32 lose what matters), and the definitions in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def listed():
    def delta(name, S, T, hk, hv, dk, dv, dtype, l2norm=True, ragged=False):
        return {"name": name, "op": "delta", "S": S, "T": T, "hk": hk, "hv": hv, "dk": dk, "dv": dv, "dtype": dtype,
                "l2norm": l2norm, "ragged": ragged}

    def norm(name, rows, groups, dim, dtype, res, post, act, pre, bias=False):
        return {"name": name, "op": "norm", "rows": rows, "groups": groups, "dim": dim, "dtype": dtype, "res": res,
                "post": post, "act": act, "pre": pre, "bias": bias}

    return [
        # one stream's next frame: nothing but latency
        delta("frame of one stream", 1, 1, 4, 8, 128, 128, "bf16"),
        # the next frame of the benchmark's 8192 streams, two heads as wide as the KWS net
        delta("frame of 8192 streams", 8192, 1, 2, 2, 64, 64, "bf16"),
        # the next frame of a wide layer, key heads shared by two value heads
        delta("frame of a wide layer", 128, 1, 16, 32, 128, 128, "bf16"),
        # the benchmark's chunk: 100 frames of 8192 streams
        delta("100 frames of 8192 streams", 8192, 100, 2, 2, 64, 64, "f16"),
        # a batch of utterances of different lengths, padded; head width of the S2I net (72)
        delta("ragged utterances", 24, 1000, 8, 16, 72, 128, "bf16", True, True),
        # a recording of minutes in one call: few rows, a long axis
        delta("long recording", 1, 16384, 16, 32, 128, 128, "bf16"),
        # 32 bits throughout, keys normalised by the caller, an odd length
        delta("777 frames in 32 bits", 16, 777, 4, 4, 64, 128, "f32", False),
        # after a block, before the next: one stream's next frame
        norm("norms of one frame", 1, 1, 1024, "bf16", "bf16", "rms", "sigmoid", "rms"),
        # the gated norm of the delta rule's heads, the benchmark's chunk
        norm("gated norm of heads", 819200, 2, 64, "bf16", "none", "rms", "silu", "none"),
        # between two blocks of a wide net, residual kept in 32 bits
        norm("norms between wide blocks", 8192, 1, 4096, "bf16", "f32", "rms", "none", "rms"),
        # layer norms with biases at an odd width
        norm("layer norms, odd width", 5000, 1, 1001, "f16", "f16", "layer", "sigmoid", "layer", True),
        # 32 bits, plain pre-norm of a residual stream
        norm("norms in 32 bits", 16384, 1, 2048, "f32", "f32", "none", "silu", "rms"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.65:
        hk = rng.choice([1, 2, 3, 4, 8, 16])
        hv = hk * rng.choice([1, 1, 2, 4])
        wide = lambda: rng.choice([rng.randint(8, 128), 4 * rng.randint(4, 32), 64, 72, 128, 8 * rng.randint(16, 32)])  # noqa: E731
        dk, dv = wide(), wide()
        T = 1 if rng.random() < 0.35 else _log(rng, 2, 16384)
        # at most half the elements of the longest recording's work, and states of at most 1 GB in all
        most = min(16384 * 32 * 128 * 128 // (2 * T * hv * dk * dv), 2 ** 28 // (hv * dk * dv))
        S = _log(rng, 1, max(1, min(8192, most)))
        while T > 1 and S * T * hv * dk * dv > 16384 * 32 * 128 * 128:
            T = max(2, T // 2)
        return {"op": "delta", "S": S, "T": T, "hk": hk, "hv": hv, "dk": dk, "dv": dv,
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "l2norm": rng.random() < 0.7,
                "ragged": T > 1 and rng.random() < 0.4}
    dim = rng.choice([rng.randint(16, 256), _log(rng, 16, 8192), 128 * rng.randint(1, 16)])
    groups = rng.choice([1, 1, 2, 8])
    rows = _log(rng, 1, max(1, min(400000, 8192 * 4096 // (dim * groups))))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    return {"op": "norm", "rows": rows, "groups": groups, "dim": dim, "dtype": dtype,
            "res": rng.choice(["none", dtype, "f32"]), "post": rng.choice(["none", "rms", "layer"]),
            "act": rng.choice(["none", "sigmoid", "silu"]), "pre": rng.choice(["rms", "rms", "layer"]),
            "bias": rng.random() < 0.3}


def _lens(c):
    """Frames per stream: the same for every seed, so that work() knows them."""
    if not c["ragged"]:
        return [c["T"]] * c["S"]
    r = random.Random(c["S"] * 100003 + c["T"])
    return [r.randint(0, c["T"]) for _ in range(c["S"] - 1)] + [c["T"]]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    if c["op"] == "norm":
        shape = (c["rows"], c["groups"], c["dim"])
        s = {"case": c, "x": (1.5 * randn(*shape)).to(dt), "y": torch.zeros(shape, dtype=dt, device="cuda"),
             "gate": randn(*shape).to(dt) if c["act"] != "none" else None, "res_in": None, "res_out": None,
             "w_post": 1 + 0.1 * randn(c["dim"]) if c["post"] != "none" else None,
             "w_pre": 1 + 0.1 * randn(c["dim"]) if c["pre"] != "none" else None,
             "b_post": 0.1 * randn(c["dim"]) if c["bias"] and c["post"] != "none" else None,
             "b_pre": 0.1 * randn(c["dim"]) if c["bias"] and c["pre"] != "none" else None, "scale": 0.5}
        if c["res"] != "none":
            s["res_in"] = (2 * randn(*shape)).to(DTYPES[c["res"]])
            s["res_out"] = torch.zeros_like(s["res_in"])
        if own:
            from nnsp_amd.seq import BlockNorm
            s["plan"] = BlockNorm(c["rows"], c["dim"], groups=c["groups"], dtype=c["dtype"],
                                  res_dtype=c["dtype"] if c["res"] == "none" else c["res"], post=c["post"],
                                  act=c["act"], pre=c["pre"], res_scale=s["scale"], eps=EPS)
        return s
    S, T, hk, hv, dk, dv = (c[n] for n in ("S", "T", "hk", "hv", "dk", "dv"))
    # keys of neighbouring frames are alike, as those of speech are
    k = randn(S, T, hk, dk) + randn(S, 1, hk, dk)
    if not c["l2norm"]:
        k = k / k.square().sum(-1, keepdim=True).sqrt()
    q = randn(S, T, hk, dk)
    if not c["l2norm"]:
        q = q / q.square().sum(-1, keepdim=True).sqrt()
    # decay per frame e^g: heads from slow (0.999) to fast (0.4)
    rate = torch.exp(torch.empty(hv, device="cuda").uniform_(-5.0, 0.0, generator=gen))
    g = -rate * torch.nn.functional.softplus(randn(S, T, hv))
    s = {"case": c, "q": q.to(dt), "k": k.to(dt), "v": randn(S, T, hv, dv).to(dt), "g": g,
         "beta": torch.sigmoid(randn(S, T, hv)), "state_in": 0.3 * randn(S, hv, dk, dv),
         "out": torch.zeros(S, T, hv, dv, dtype=dt, device="cuda"),
         "state_out": torch.zeros(S, hv, dk, dv, device="cuda"),
         "lens": torch.tensor(_lens(c), dtype=torch.int32, device="cuda") if c["ragged"] else None}
    if own:
        from nnsp_amd.seq import GatedDelta
        s["plan"] = GatedDelta(S, T, hk, hv, dk, dv, dtype=c["dtype"], l2norm=c["l2norm"], eps=EPS)
        n = s["plan"].workspace_bytes
        s["workspace"] = torch.empty(n, dtype=torch.uint8, device="cuda") if n else None
    return s


def _ptr(t):
    return None if t is None else t.data_ptr()


def run(state):
    s, c = state, state["case"]
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        if c["op"] == "norm":
            s["plan"].exec_device(_ptr(s["x"]), _ptr(s["y"]), gate=_ptr(s["gate"]), w_post=_ptr(s["w_post"]),
                                  b_post=_ptr(s["b_post"]), w_pre=_ptr(s["w_pre"]), b_pre=_ptr(s["b_pre"]),
                                  res_in=_ptr(s["res_in"]), res_out=_ptr(s["res_out"]), stream=stream)
            return {"y": s["y"], "res_out": s["res_out"]}
        s["plan"].exec_device(_ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["g"]), _ptr(s["beta"]), _ptr(s["out"]),
                              state_in=_ptr(s["state_in"]), state_out=_ptr(s["state_out"]), lens=_ptr(s["lens"]),
                              workspace=_ptr(s["workspace"]), stream=stream)
        return {"out": s["out"], "state": s["state_out"]}
    if c["op"] == "norm":
        y, r = _plain_norm(s, c)
        return {"y": y.to(s["y"].dtype), "res_out": None if s["res_in"] is None else r.to(s["res_in"].dtype)}
    out, S1 = _plain_delta(s, c)
    out = out.to(s["out"].dtype)
    if s["lens"] is not None:
        frames = torch.arange(c["T"], device="cuda")
        out = torch.where((frames[None, :] < s["lens"][:, None])[..., None, None], out, s["out"])
    return {"out": out, "state": S1}


def _normed(x, kind, w, b):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    return x if b is None else x + b


def _plain_norm(s, c):
    h = _normed(s["x"].float(), c["post"], s["w_post"], s["b_post"])
    if c["act"] != "none":
        z = s["gate"].float()
        gate = 1 / (1 + torch.exp(-z))
        h = h * (gate if c["act"] == "sigmoid" else z * gate)
    r = s["scale"] * h
    if s["res_in"] is not None:
        r = s["res_in"].float() + r
    return _normed(r, c["pre"], s["w_pre"], s["b_pre"]), r


def _unit_lower_inverse(A):
    """(I + A)^-1 of strictly lower A [..., C, C], C a power of two: blocks of 1, 2, 4, ... joined pairwise by
    [[a, 0], [x, d]]^-1 = [[a^-1, 0], [-d^-1 x a^-1, d^-1]]."""
    C, n = A.shape[-1], 1
    inv = torch.ones(A.shape[:-2] + (C, 1, 1), dtype=A.dtype, device=A.device)
    while n < C:
        blocks = A.reshape(A.shape[:-2] + (C // (2 * n), 2, n, C // (2 * n), 2, n))
        at = torch.arange(C // (2 * n), device=A.device)
        x = blocks[..., at, 1, :, at, 0, :].movedim(0, -3)
        a, d = inv[..., 0::2, :, :], inv[..., 1::2, :, :]
        x = -(d @ (x @ a))
        inv = torch.cat([torch.cat([a, torch.zeros_like(a)], -1), torch.cat([x, d], -1)], -2)
        n *= 2
    return inv.squeeze(-3)


def _plain_delta(s, c):
    S, T, hk, hv, dk, dv = (c[n] for n in ("S", "T", "hk", "hv", "dk", "dv"))
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["l2norm"]:
        q = q * torch.rsqrt(q.square().sum(-1, keepdim=True) + EPS)
        k = k * torch.rsqrt(k.square().sum(-1, keepdim=True) + EPS)
    q = q * dk ** -0.5
    g, beta = s["g"], s["beta"]
    if s["lens"] is not None:
        live = (torch.arange(T, device="cuda")[None, :] < s["lens"][:, None])[..., None]
        g, beta = torch.where(live, g, 0), torch.where(live, beta, 0)
    C = 1
    while C < min(T, 64):
        C *= 2
    N = -(-T // C)

    def chunks(x, heads):  # [S, T, heads, d] -> [S * hv, N, C, d]
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, N * C - T))
        x = x.repeat_interleave(hv // heads, 2) if heads != hv else x
        return x.movedim(2, 1).reshape(S * hv, N, C, -1)

    q, k, v = chunks(q, hk), chunks(k, hk), chunks(v, hv)
    g, beta = chunks(g[..., None], hv)[..., 0], chunks(beta[..., None], hv)
    G = g.double().cumsum(-1)
    decay = torch.exp((G[..., :, None] - G[..., None, :]).clamp(max=0)).float()
    up, rest, whole = torch.exp(G).float()[..., None], torch.exp(G[..., -1:] - G).float()[..., None], torch.exp(G[..., -1]).float()
    T_ = _unit_lower_inverse(torch.tril(beta * (k @ k.mT) * decay, -1))
    P = torch.tril((q @ k.mT) * decay)
    U0, W = T_ @ (beta * v), T_ @ (beta * up * k)
    q, kr = q * up, (k * rest).mT
    state, out = s["state_in"].reshape(S * hv, dk, dv), torch.empty_like(v)
    for n in range(N):
        U = U0[:, n] - W[:, n] @ state
        out[:, n] = q[:, n] @ state + P[:, n] @ U
        state = whole[:, n, None, None] * state + kr[:, n] @ U
    out = out.reshape(S, hv, N * C, dv)[:, :, :T].movedim(1, 2)
    return out, state.reshape(S, hv, dk, dv)


def work(case):
    c = case
    if c["op"] == "norm":
        n = c["rows"] * c["groups"] * c["dim"]
        size = DTYPES[c["dtype"]].itemsize
        per = 2 * size + (size if c["act"] != "none" else 0)
        per += 2 * DTYPES[c["res"]].itemsize if c["res"] != "none" else 0
        return {"bytes": n * per + 4 * c["dim"] * ((c["post"] != "none") + (c["pre"] != "none")) * (2 if c["bias"] else 1),
                "flops": 12 * n}
    frames, size = sum(_lens(c)), DTYPES[c["dtype"]].itemsize
    per = size * (2 * c["hk"] * c["dk"] + 2 * c["hv"] * c["dv"]) + 8 * c["hv"]
    return {"bytes": frames * per + 8 * c["S"] * c["hv"] * c["dk"] * c["dv"] + (4 * c["S"] if c["ragged"] else 0),
            "flops": 6 * frames * c["hv"] * c["dk"] * c["dv"]}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    d = {n: t.double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for n, t in s.items()}
    if case["op"] == "norm":
        def norm(x, kind, w, b):
            if kind == "none":
                return x
            mean = x.mean(-1, keepdim=True) if kind == "layer" else 0.0
            var = ((x - mean) ** 2).sum(-1, keepdim=True) / x.shape[-1]
            x = (x - mean) / (var + EPS).sqrt() * w
            return x if b is None else x + b

        h = norm(d["x"], case["post"], d["w_post"], d["b_post"])
        if case["act"] == "sigmoid":
            h = h * torch.sigmoid(d["gate"])
        elif case["act"] == "silu":
            h = h * d["gate"] * torch.sigmoid(d["gate"])
        r = d["scale"] * h + (0 if d["res_in"] is None else d["res_in"])
        return {"y": norm(r, case["pre"], d["w_pre"], d["b_pre"]), "res_out": None if d["res_in"] is None else r}
    # frame by frame, as the rule is written
    S, T, hk, hv, dk = (case[n] for n in ("S", "T", "hk", "hv", "dk"))
    of = torch.arange(hv, device="cuda") // (hv // hk)
    state, out = d["state_in"].clone(), torch.zeros_like(d["out"])
    lens = None if d["lens"] is None else d["lens"].long()
    for t in range(T):
        q, k = d["q"][:, t, of], d["k"][:, t, of]
        if case["l2norm"]:
            q = q / ((q * q).sum(-1, keepdim=True) + EPS).sqrt()
            k = k / ((k * k).sum(-1, keepdim=True) + EPS).sqrt()
        new = state * torch.exp(d["g"][:, t])[..., None, None]
        u = d["beta"][:, t, :, None] * (d["v"][:, t] - (new * k[..., None]).sum(-2))
        new = new + k[..., None] * u[..., None, :]
        o = (new * q[..., None]).sum(-2) * dk ** -0.5
        if lens is None:
            state, out[:, t] = new, o
        else:
            live = (t < lens)[:, None, None]
            state, out[:, t] = torch.where(live[..., None], new, state), torch.where(live, o, 0.0)
    return {"out": out, "state": state}
