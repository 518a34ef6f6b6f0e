"""Cases, plain forms and 64-bit forms of the operators of a LoRA training step on a microscaled 4-bit base.

    residual   r = residual_scale * x + gate * post(y);  z = norm(r) * (1 + scale) + shift
               (the norm after a sub-block, its gate and residual scale, and the norm before the next)
    prenorm    z = zrms(x) * (1 + scale) + shift
    gradnorm   the 2-norm of many gradient tensors taken as one vector
    clip       the same norm, and every tensor times min(1, max_norm / (norm + 1e-6))
    quantise   blocks of 32 values along a row as 4-bit floats (e2m1) under one power-of-two scale (e8m0)
    linear     y = dequant(quant(x)) . dequant(W)^T + bias, and dx = dy . dequant(W)

`own` chooses the side: False runs the plain forms below, True the calls of `loractl_b200`.
"""
import torch

own = False

DEV = "cuda"
EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # the trunk at its published width: one 512-pixel sample, between attention and the MLP, training
        {"name": "residual_train_wide", "op": "residual", "b": 1, "t": 1536, "h": 6144, "dtype": "bf16", "mod": "bf16",
         "norm": "zrms", "post": False, "alpha": 1.0, "train": True},
        # a batch of image streams with layer norms, training: the longest pass over activations
        {"name": "residual_train_batch", "op": "residual", "b": 8, "t": 4096, "h": 2048, "dtype": "bf16", "mod": "bf16",
         "norm": "layer", "post": False, "alpha": 1.0, "train": True},
        # text tokens of one prompt with a norm behind the sub-block too, no gradient: latency
        {"name": "residual_infer_text", "op": "residual", "b": 1, "t": 77, "h": 6144, "dtype": "bf16", "mod": "f32",
         "norm": "zrms", "post": True, "alpha": 0.5, "train": False},
        # odd width and lengths in f32 (reference numerics), every gradient, trained norm weights
        {"name": "residual_train_odd", "op": "residual", "b": 3, "t": 333, "h": 1155, "dtype": "f32", "mod": "f32",
         "norm": "zrms", "post": True, "alpha": 0.75, "train": True},
        # every LoRA factor of a 28-block trunk at rank 16: 392 tensors, more than the L2 holds
        {"name": "gradnorm_trunk", "op": "gradnorm", "layers": 28, "rank": 16, "width": 6144, "inner": 16384, "dtype": "f32"},
        # a text model's factors at rank 8: 96 small tensors, latency
        {"name": "clip_text_model", "op": "clip", "layers": 12, "rank": 8, "width": 768, "inner": 2048, "dtype": "f32",
         "max_norm": 1.0},
        # gradients kept in both types, odd widths
        {"name": "clip_mixed_odd", "op": "clip", "layers": 9, "rank": 33, "width": 5001, "inner": 7777, "dtype": "mixed",
         "max_norm": 0.5},
        # activations of one trunk sample
        {"name": "quantise_trunk", "op": "quantise", "n": 1536, "k": 16384, "dtype": "bf16"},
        # a short ragged f32 batch
        {"name": "quantise_odd", "op": "quantise", "n": 333, "k": 1184, "dtype": "f32"},
        # the conditioning vector of one sample through a wide projection: the weight's bytes are the work
        {"name": "linear_one_token", "op": "linear", "n": 1, "k": 6144, "m": 16384, "dtype": "bf16", "bias": True, "train": False},
        # text tokens through an odd projection in f32
        {"name": "linear_text_odd", "op": "linear", "n": 77, "k": 2592, "m": 6151, "dtype": "f32", "bias": True, "train": False},
        # two trunk samples through the up-projection with the input's gradient: the matrix products are the work
        {"name": "linear_train_wide", "op": "linear", "n": 4096, "k": 6144, "m": 16384, "dtype": "bf16", "bias": False, "train": True},
    ]


def _log(rng, lo, hi):
    import math
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["residual", "residual", "prenorm", "gradnorm", "clip", "quantise", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("residual", "prenorm"):
        h = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            h = max(64, h // 64 * 64)
        b = _log(rng, 1, 8)
        t = _log(rng, 1, max(2, (1 << 25) // (b * h)))
        case = {"op": op, "b": b, "t": t, "h": h, "dtype": dtype, "mod": rng.choice(["f32", dtype]), "train": rng.random() < 0.6}
        if op == "residual":
            case.update(norm=rng.choice(["zrms", "layer"]), post=rng.random() < 0.4, alpha=rng.choice([1.0, 0.5, 0.8125]))
        return case
    if op in ("gradnorm", "clip"):
        case = {"op": op, "layers": _log(rng, 1, 28), "rank": _log(rng, 1, 24), "width": _log(rng, 32, 4096),
                "inner": _log(rng, 64, 8192), "dtype": rng.choice(["f32", "bf16", "mixed"])}
        if op == "clip":
            case["max_norm"] = rng.choice([0.1, 1.0, 1e6])
        return case
    k = 32 * _log(rng, 1, 512)
    if op == "quantise":
        return {"op": op, "n": _log(rng, 1, max(2, (1 << 24) // k)), "k": k, "dtype": dtype}
    n, m = _log(rng, 1, 4096), _log(rng, 8, 16384)
    if dtype == "f32":  # reference numerics is a small-model path
        k, n, m = min(k, 4096), min(n, 512), min(m, 4096)
    n = min(n, max(1, (1 << 38) // (m * k)))
    return {"op": op, "n": n, "k": k, "m": m, "dtype": dtype, "bias": rng.random() < 0.5, "train": rng.random() < 0.5}


# ---- inputs -----------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _activations(g, shape):
    """Unit-variance tokens with a few channels an order of magnitude larger, as trained blocks have."""
    x = torch.randn(shape, generator=g, device=DEV)
    big = torch.rand(shape[-1], generator=g, device=DEV) < 0.01
    return x * torch.where(big, 12.0, 1.0)


def _factor_shapes(case):
    r, w, i = case["rank"], case["width"], case["inner"]
    kv = max(1, w // 4)
    sites = [(w, w), (w, kv), (w, kv), (w, w), (w, i), (w, i), (i, w)]
    return [s for _ in range(case["layers"]) for d_in, d_out in sites for s in ((d_in, r), (r, d_out))]


def _bucket(case, grads):
    """One zeroed flat buffer for each type and a view of it for each tensor, 64 elements apart at least as the
    adapters' bucket has them; back to back for the odd case."""
    gap = 1 if case["dtype"] == "mixed" else 64
    ends, at = {}, []
    for v in grads:
        lo = -(-ends.get(v.dtype, 0) // gap) * gap
        at.append(lo)
        ends[v.dtype] = lo + v.numel()
    flat = {dt: torch.zeros(n, dtype=dt, device=DEV) for dt, n in ends.items()}
    return list(flat.values()), [flat[v.dtype][lo:lo + v.numel()].view(v.shape) for v, lo in zip(grads, at)]


def prepare(case, seed):
    g = _gen(seed)
    op, st = case["op"], {"case": case}
    if op in ("residual", "prenorm"):
        b, t, h = case["b"], case["t"], case["h"]
        dt, mt = TYPES[case["dtype"]], TYPES[case["mod"]]
        x = _activations(g, (b, t, h))
        y = torch.randn((b, t, h), generator=g, device=DEV)
        pad = t // 8  # a sequence is padded with zero tokens up to its length
        if pad:
            x[:, t - pad:] = 0
            y[:, t - pad:] = 0
        mod = torch.randn((b, 1, 3 * h), generator=g, device=DEV) * 0.3
        shift, scale, gate = mod.to(mt).chunk(3, dim=-1)  # slices of one modulation tensor, as a block has them
        st.update(x=x.to(dt), y=y.to(dt), shift=shift, scale=scale, gate=gate)
        st["weight"] = torch.randn(h, generator=g, device=DEV) * 0.2
        st["post_weight"] = torch.randn(h, generator=g, device=DEV) * 0.2
        st["dr"] = (torch.randn((b, t, h), generator=g, device=DEV) * 0.1).to(dt)
        st["dz"] = (torch.randn((b, t, h), generator=g, device=DEV) * 0.1).to(dt)
        if op == "prenorm":
            names = ["x", "weight", "shift", "scale"]
        else:
            names = ["x", "gate", "y", "shift", "scale"]
            names += ["weight"] if case["norm"] == "zrms" else []
            names += ["post_weight"] if case["post"] else []
        st["names"] = names
        if case["train"]:
            for n in names:
                st[n] = st[n].detach().requires_grad_(True)
    elif op in ("gradnorm", "clip"):
        grads = []
        for i, shape in enumerate(_factor_shapes(case)):
            dt = torch.bfloat16 if case["dtype"] == "bf16" or (case["dtype"] == "mixed" and i % 3 == 1) else torch.float32
            size = 10.0 ** (-2 - 2 * (i % 5) / 5)  # layers differ by orders of magnitude
            grads.append((torch.randn(shape, generator=g, device=DEV) * size).to(dt))
        st["grads"] = grads
        if op == "clip":
            st["flat"], st["out"] = _bucket(case, grads)
    else:
        n, k, dt = case["n"], case["k"], TYPES[case["dtype"]]
        st["x"] = _activations(g, (n, k)).to(dt)
        if op == "linear":
            m = case["m"]
            w = (torch.randn((m, k), generator=g, device=DEV) * 0.02).to(torch.bfloat16)
            st["bias"] = torch.randn(m, generator=g, device=DEV) * 0.1 if case["bias"] else None
            st["dy"] = (torch.randn((n, m), generator=g, device=DEV) * 0.1).to(dt)
            if own:
                import loractl_b200 as lb
                st["layer"] = lb.Mx4Linear(lb.mx4_quantize(w), st["bias"])
            else:
                codes, exps = _codes(w.float())
                st["w"] = (codes, exps)
            if case["train"]:
                st["x"].requires_grad_(True)
    return st


# ---- one pass ---------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import loractl_b200 as lb

    case, op = s["case"], s["case"]["op"]
    if op in ("residual", "prenorm"):
        if op == "prenorm":
            outs, dys = (lb.block_ops.modulated_zrmsnorm(s["x"], s["weight"], s["shift"], s["scale"]),), (s["dz"],)
        else:
            outs = lb.block_ops.gated_residual_norm(
                s["x"], s["gate"], s["y"], s["shift"], s["scale"], norm=case["norm"], residual_scale=case["alpha"],
                weight=s["weight"] if case["norm"] == "zrms" else None, post_weight=s["post_weight"] if case["post"] else None)
            dys = (s["dr"], s["dz"])
        if not case["train"]:
            return tuple(outs)
        grads = torch.autograd.grad(outs, [s[n] for n in s["names"]], dys)
        return tuple(o.detach() for o in outs) + tuple(grads)
    if op == "gradnorm":
        return lb.global_grad_norm(s["grads"])
    if op == "clip":
        norm = lb.clip_grad_norm(s["grads"], case["max_norm"], out=s["out"])
        return [norm] + s["flat"]
    if op == "quantise":
        return lb.mx4_quantize(s["x"]).dequantize(s["x"].dtype)
    y = s["layer"](s["x"])
    if not case["train"]:
        return y
    return y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]


def _run_plain(s):
    case, op = s["case"], s["case"]["op"]
    if op in ("residual", "prenorm"):
        x, dt = s["x"].float(), s["x"].dtype
        if op == "prenorm":
            r = x
        else:
            y = s["y"].float()
            if case["post"]:
                y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * (1 + s["post_weight"])
            r = case["alpha"] * x + s["gate"].float() * y
        if op == "prenorm" or case["norm"] == "zrms":
            z = r / torch.sqrt((r * r).mean(-1, keepdim=True) + EPS) * (1 + s["weight"])
        else:
            c = r - r.mean(-1, keepdim=True)
            z = c / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
        z = z * (1 + s["scale"].float()) + s["shift"].float()
        outs = (z.to(dt),) if op == "prenorm" else (r.to(dt), z.to(dt))
        if not case["train"]:
            return outs
        dys = (s["dz"],) if op == "prenorm" else (s["dr"], s["dz"])
        grads = torch.autograd.grad(outs, [s[n] for n in s["names"]], dys)
        return tuple(o.detach() for o in outs) + tuple(grads)
    if op in ("gradnorm", "clip"):
        total = torch.zeros((), dtype=torch.float64, device=DEV)
        for v in s["grads"]:
            d = v.double()
            total = total + (d * d).sum()
        norm = torch.sqrt(total)
        if op == "gradnorm":
            return norm.float()
        coef = torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0).float()
        for v, o in zip(s["grads"], s["out"]):
            o.copy_(v.float() * coef)
        return [norm.float()] + s["flat"]
    if op == "quantise":
        return _values(*_codes(s["x"].float())).to(s["x"].dtype)
    x, dt = s["x"], s["x"].dtype
    w = _values(*s["w"])
    y = _values(*_codes(x.detach().float())) @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    y = y.to(dt)
    if not case["train"]:
        return y
    return y, (s["dy"].float() @ w).to(dt)


def _power(e):
    """2^e in f32 from its bits, e in [-127, 128] (128 stands for the NaN of the scale's type)."""
    bits = (e.to(torch.int32) + 127) << 23
    bits = torch.where(e == -127, torch.full_like(bits, 0x00400000), bits)
    bits = torch.where(e == 128, torch.full_like(bits, 0x7FC00000), bits)
    return bits.view(torch.float32)


def _codes(x):
    """f32 [n, k] -> (signed multiples of the scale, [n, k / 32, 32] int8 in halves; exponents [n, k / 32])."""
    n, k = x.shape
    v = x.reshape(n, k // 32, 32)
    top = v.abs().amax(-1)
    e = (torch.frexp(top)[1] - 3).clamp(-127, 125)
    e = torch.where(top == 0, torch.full_like(e, -127), e)
    s = v.abs() * _power(-e).unsqueeze(-1)
    step = torch.where(s < 2, 0.5, torch.where(s < 4, 1.0, 2.0))
    q = (torch.round(s / step) * step).clamp(max=6.0)
    q = torch.where(v < 0, -q, q)
    bad = ~torch.isfinite(v).all(-1)
    e = torch.where(bad, torch.full_like(e, 128), e)
    return torch.where(bad.unsqueeze(-1), 0.0, 2 * q).to(torch.int8), e.to(torch.int16)


def _values(codes, e):
    n, blocks, _ = codes.shape
    return (codes.float() * 0.5 * _power(e).unsqueeze(-1)).reshape(n, blocks * 32)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    op = case["op"]
    size = lambda key: 4 if case[key] == "f32" else 2
    if op in ("residual", "prenorm"):
        e, m = case["b"] * case["t"] * case["h"], case["b"] * case["h"]
        two = op == "residual"
        vec = (3 if two else 2) * m * size("mod") + 2 * 4 * case["h"]
        fwd = e * size("dtype") * (4 if two else 2) + vec          # x (y) in, (r) z out
        bwd = e * size("dtype") * (4 if two else 2) + vec          # (dr) dz in, dx (dy) out
        return {"bytes": fwd + (bwd if case["train"] else 0), "flops": e * (40 if case["train"] else 14)}
    if op in ("gradnorm", "clip"):
        bytes_, count = 0, 0
        for i, (a, b) in enumerate(_factor_shapes(case)):
            count += a * b
            bytes_ += a * b * (2 if case["dtype"] == "bf16" or (case["dtype"] == "mixed" and i % 3 == 1) else 4)
        return {"bytes": bytes_ * (2 if op == "clip" else 1), "flops": count * (3 if op == "clip" else 2)}
    n, k = case["n"], case["k"]
    if op == "quantise":
        return {"bytes": 2 * n * k * size("dtype"), "flops": 6 * n * k}
    m = case["m"]
    w = m * k // 2 + m * k // 32
    act = (n * k + n * m) * size("dtype") + (4 * m if case["bias"] else 0)
    if not case["train"]:
        return {"bytes": w + act, "flops": 2 * n * m * k}
    return {"bytes": w + 2 * act, "flops": 4 * n * m * k}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op in ("residual", "prenorm"):
        return _exact_norm(case, s)
    if op in ("gradnorm", "clip"):
        flat = torch.cat([v.reshape(-1).to(torch.float64) for v in s["grads"]])
        norm = torch.linalg.vector_norm(flat)
        if op == "gradnorm":
            return norm
        f = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
        for v, o in zip(s["grads"], s["out"]):  # marks the places; the values are formed in 64 bits below
            o.copy_(v)
        return [norm] + [v.double() * f for v in s["flat"]]
    x = s["x"].detach().double()
    xq = _nearest(x)
    if op == "quantise":
        return xq
    g = _gen(seed)
    _activations(g, (case["n"], case["k"]))
    w = (torch.randn((case["m"], case["k"]), generator=g, device=DEV) * 0.02).to(torch.bfloat16).double()
    w = _nearest(w)
    y = torch.einsum("nk,mk->nm", xq, w)
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if not case["train"]:
        return y
    return y, torch.einsum("nm,mk->nk", s["dy"].double(), w)


def _nearest(x):
    """Nearest value of {0, .5, 1, 1.5, 2, 3, 4, 6} times the block's power of two, ties to the even code."""
    n, k = x.shape
    v = x.reshape(-1, 32)
    top = v.abs().max(dim=1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    low = torch.exp2(e)
    e = torch.where(low > top, e - 1, torch.where(2 * low <= top, e + 1, e)) - 2
    unit = torch.exp2(torch.where(top > 0, e, torch.full_like(e, -127.0)).clamp(-127, 125))
    a = v.abs() / unit
    out = torch.zeros_like(a)
    # (border, value above it, whether the border itself goes up)
    for border, value, up in ((0.25, 0.5, False), (0.75, 1.0, True), (1.25, 1.5, False), (1.75, 2.0, True),
                              (2.5, 3.0, False), (3.5, 4.0, True), (5.0, 6.0, False)):
        out = torch.where((a >= border) if up else (a > border), torch.full_like(out, value), out)
    out = torch.copysign(out, v) * unit
    return torch.where(torch.isfinite(top), out, torch.full_like(out, float("nan"))).reshape(n, k)


def _exact_norm(case, s):
    d = lambda name: s[name].detach().double()
    two = case["op"] == "residual"
    post = two and case["post"]
    zrms = not two or case["norm"] == "zrms"
    x, shift, scale = d("x"), d("shift"), d("scale")
    alpha = case["alpha"] if two else 1.0
    h = case["h"]
    weight = d("weight") if zrms else torch.zeros(h, dtype=torch.float64, device=DEV)
    if two:
        y, gate = d("y"), d("gate")
        prs = (y.square().sum(-1, keepdim=True) / h + EPS).rsqrt() if post else None
        yh = y * prs if post else y
        pw = 1 + d("post_weight") if post else 1.0
        r = alpha * x + gate * (yh * pw)
    else:
        r = x
    mu = 0.0 if zrms else r.sum(-1, keepdim=True) / h
    rs = ((r - mu).square().sum(-1, keepdim=True) / h + EPS).rsqrt()
    rh = (r - mu) * rs
    z = rh * (1 + weight) * (1 + scale) + shift
    outs = (r, z) if two else (z,)
    if not case["train"]:
        return outs
    dz = d("dz")
    g = dz * (1 + weight) * (1 + scale)
    back = g - rh * (g * rh).mean(-1, keepdim=True)
    if not zrms:
        back = back - g.mean(-1, keepdim=True)
    dr = rs * back + (d("dr") if two else 0.0)
    shape = lambda v, name: v.reshape(s[name].shape)
    sums = (dz * rh).sum(1, keepdim=True)
    grads = {"x": alpha * dr, "shift": shape(dz.sum(1, keepdim=True), "shift"), "scale": shape(sums * (1 + weight), "scale"),
             "weight": (sums * (1 + scale)).sum((0, 1))}
    if two:
        du = gate * dr
        grads["gate"] = shape((dr * yh * pw).sum(1, keepdim=True), "gate")
        if post:
            grads["post_weight"] = (du * yh).sum((0, 1))
            dyh = du * pw
            grads["y"] = prs * (dyh - yh * (dyh * yh).mean(-1, keepdim=True))
        else:
            grads["y"] = du
    return outs + tuple(grads[n] for n in s["names"])
