"""`gated_residual_norm` / `modulated_zrmsnorm` (crates/loractl-core/src/mmdit.rs:282-330,857-869 in one pass) against
the formulas in 64 bits: values and every gradient, both norms, with and without the norm behind the sub-block, odd
widths and lengths, strided and broadcast inputs, zero rows, and the calls that are refused.

Tolerances, for values relative to the largest of the tensor: an output held in bf16 is off by at most half a step of
its own value (2^-9 of the largest is reached by values in the upper half of a binade, 2^-8 bounds all) plus the f32
arithmetic; f32 arithmetic along a row of h <= 16384 elements and a sum over n tokens adds up in trees and
runs of at most max(32, rows of one chunk) terms, each off by 2^-24 of a partial sum, so 2^-24 * 64 = 4e-6 of the
largest magnitude that is summed; sums that cancel are measured by the sum of their terms' magnitudes."""
import pytest
import torch

EPS = 1e-5
SHAPES = [(1, 1, 64), (2, 5, 96), (1, 77, 6144), (3, 129, 521), (2, 300, 1155), (1, 33, 8200), (1, 5, 16384), (40, 1, 72), (1, 1, 1),
          (700, 3, 40)]


def make(b, t, h, dtype, mod, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda")
    v = {"x": (mk(b, t, h) * 1.5 + 0.3).to(dtype), "y": mk(b, t, h).to(dtype)}
    mods = mk(b, 1, 3 * h).to(mod) * 0.4
    v["gate"], v["shift"], v["scale"] = mods.chunk(3, dim=-1)
    v["weight"], v["post_weight"] = mk(h) * 0.3, mk(h) * 0.3
    v["dr"], v["dz"] = mk(b, t, h).to(dtype), mk(b, t, h).to(dtype)
    return v


def formula(v, norm, post, alpha, two=True):
    """r and z in 64 bits from 64-bit leaves, by elementary operations."""
    if two:
        y = v["y"]
        if post:
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * (1 + v["post_weight"])
        r = alpha * v["x"] + v["gate"].reshape(v["x"].shape[0], 1, -1) * y
    else:
        r = v["x"]
    c = r - r.mean(-1, keepdim=True) if norm == "layer" else r
    n = c / (c.square().mean(-1, keepdim=True) + EPS).sqrt()
    if v.get("weight") is not None:
        n = n * (1 + v["weight"])
    b = r.shape[0]
    return r, n * (1 + v["scale"].reshape(b, 1, -1)) + v["shift"].reshape(b, 1, -1)


def close(ours, ref, dtype, summed=None, what=""):
    assert ours.shape == ref.shape and ours.dtype == dtype, what
    top = float((summed if summed is not None else ref).abs().max()) if ref.numel() else 0.0
    err = (ours.double() - ref).abs()
    tol = 4e-6 * top + (2.0 ** -8 * ref.abs() if dtype == torch.bfloat16 else 2.0 ** -23 * ref.abs())
    assert bool((err <= tol + 1e-30).all()), f"{what}: {float((err - tol).max()):.3e} over at a largest of {top:.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("b,t,h", SHAPES)
@pytest.mark.parametrize("dtype,mod", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                       (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("norm,post,alpha", [("zrms", False, 1.0), ("layer", False, 0.5), ("zrms", True, 0.8125), ("layer", True, 1.0)])
def test_values_and_gradients_match_the_formulas(b, t, h, dtype, mod, norm, post, alpha):
    from loractl_b200.block_ops import gated_residual_norm

    v = make(b, t, h, dtype, mod)
    names = ["x", "gate", "y", "shift", "scale", "weight"] + (["post_weight"] if post else [])
    leaves = [v[n].detach().requires_grad_(True) for n in names]
    kw = dict(zip(names, leaves))
    r, z = gated_residual_norm(**kw, norm=norm, residual_scale=alpha)
    grads = torch.autograd.grad((r, z), leaves, (v["dr"], v["dz"]))
    ref = {n: v[n].detach().double().requires_grad_(True) for n in names}
    rr, rz = formula(ref, norm, post, alpha)
    rgrads = torch.autograd.grad((rr, rz), [ref[n] for n in names], (v["dr"].double(), v["dz"].double()))
    close(r, rr.detach(), dtype, what="r")
    close(z, rz.detach(), dtype, what="z")
    # dx and dy are dr + s (gz - mean(gz) - rh mean(gz rh)) times alpha or gate: in a narrow row the terms in the
    # bracket cancel (for one column gz - rh^2 gz is gz eps s^2), and each term has been rounded at 2^-24 of ITS size,
    # so the error is measured by the largest s |gz| and |dr|, not by what is left of them
    c = rr.detach() - (rr.detach().mean(-1, keepdim=True) if norm == "layer" else 0.0)
    s_row = (c.square().mean(-1, keepdim=True) + EPS).rsqrt()
    gz = v["dz"].double() * (1 + v["weight"].double()) * (1 + v["scale"].detach().double())
    terms_row = (s_row * gz).abs().max() + v["dr"].double().abs().max()
    # a token or sample sum is off by at most 4e-6 of the sum of its terms' magnitudes (D counted as above)
    rh, y = (c * s_row).abs(), v["y"].double()
    q = (y.square().mean(-1, keepdim=True) + EPS).rsqrt() if post else torch.ones_like(y[..., :1])
    pw = 1 + (v["post_weight"].double() if post else 0.0)
    dz, gate = v["dz"].double().abs(), v["gate"].detach().double().abs()
    terms = {
        "x": terms_row,
        "y": terms_row * gate.max() * ((q * (pw.abs().max())).max() if post else 1.0),
        "shift": dz.sum(1), "scale": (dz * rh * (1 + v["weight"].double()).abs()).sum(1),
        "weight": (dz * rh * (1 + v["scale"].detach().double()).abs()).sum((0, 1)),
        "gate": terms_row * (y * q * pw).abs().sum(1), "post_weight": terms_row * (y * q).abs().mul(gate).sum((0, 1)),
    }
    for n, ours, theirs in zip(names, grads, rgrads):
        close(ours, theirs.reshape(ours.shape), v[n].dtype, terms[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("b,t,h", [(1, 1, 64), (2, 33, 6144), (3, 129, 521)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("weighted", [True, False])
def test_prenorm_matches_the_formula(b, t, h, dtype, weighted):
    from loractl_b200.block_ops import modulated_zrmsnorm

    v = make(b, t, h, dtype, dtype, seed=1)
    v["weight"] = v["weight"] if weighted else None
    names = ["x", "shift", "scale"] + (["weight"] if weighted else [])
    for n in names:
        v[n] = v[n].detach().requires_grad_(True)
    z = modulated_zrmsnorm(v["x"], v["weight"], v["shift"], v["scale"])
    grads = torch.autograd.grad(z, [v[n] for n in names], v["dz"])
    ref = {n: v[n].detach().double().requires_grad_(True) for n in names}
    _, rz = formula(ref, "zrms", False, 1.0, two=False)
    close(z, rz.detach(), dtype, what="z")
    for n, ours, theirs in zip(names, grads, torch.autograd.grad(rz, [ref[n] for n in names], v["dz"].double())):
        close(ours, theirs.reshape(ours.shape), v[n].dtype, theirs.abs().max() * (t * b) ** 0.5 * 4, n)


@pytest.mark.gpu
def test_gradient_matches_differences():
    """Central differences of the f32 loss along one direction per argument: step 1e-2 (truncation, third order:
    1e-6 of the third derivative) over a loss of size ~1e2 with f32 rounding 1e-5: 1e-3 relative to the slope's scale."""
    from loractl_b200.block_ops import gated_residual_norm

    v = make(2, 7, 96, torch.float32, torch.float32, seed=2)
    names = ["x", "gate", "y", "shift", "scale", "weight", "post_weight"]
    leaves = {n: v[n].detach().clone().requires_grad_(True) for n in names}

    def loss(d):
        r, z = gated_residual_norm(**d, residual_scale=0.75)
        return (r.double() * v["dr"].double()).sum() + (z.double() * v["dz"].double()).sum()

    grads = torch.autograd.grad(loss(leaves), [leaves[n] for n in names])
    g = torch.Generator(device="cuda").manual_seed(3)
    for n, gr in zip(names, grads):
        d = torch.randn(v[n].shape, generator=g, device="cuda")
        up, down = ({**leaves, n: leaves[n].detach() + s * d} for s in (1e-2, -1e-2))
        with torch.no_grad():
            diff = float((loss(up) - loss(down)) / 2e-2)
        slope = float((gr.double() * d).sum())
        assert abs(diff - slope) <= 2e-3 * float((gr.abs() * d.abs()).sum()), n


@pytest.mark.gpu
def test_strided_broadcast_and_partial_inputs():
    """Token slices of a longer sequence, one modulation vector expanded over the samples, gradients of a sum over
    one output only, and arguments without a gradient give what the dense call gives, bit for bit."""
    from loractl_b200.block_ops import gated_residual_norm

    v = make(3, 40, 256, torch.bfloat16, torch.bfloat16, seed=4)
    one = v["gate"][:1]
    wide_x = torch.randn(3, 50, 256, device="cuda").to(torch.bfloat16)
    wide_x[:, 5:45] = v["x"]
    sx = wide_x[:, 5:45].requires_grad_(True)
    shared = one.detach().requires_grad_(True)
    r, z = gated_residual_norm(sx, shared.expand(3, 1, 256), v["y"], v["shift"], v["scale"], weight=v["weight"])
    r2, z2 = gated_residual_norm(v["x"], one.repeat(3, 1, 1), v["y"].contiguous(), v["shift"].contiguous(), v["scale"].contiguous(),
                                 weight=v["weight"])
    assert torch.equal(r, r2) and torch.equal(z, z2)
    dx, dg = torch.autograd.grad(z, (sx, shared), v["dz"])
    gd = one.repeat(3, 1, 1).requires_grad_(True)
    x2 = v["x"].clone().requires_grad_(True)
    _, z3 = gated_residual_norm(x2, gd, v["y"], v["shift"], v["scale"], weight=v["weight"])
    dx2, dg2 = torch.autograd.grad(z3, (x2, gd), v["dz"])
    assert torch.equal(dx, dx2) and torch.equal(dg, dg2.sum(0, keepdim=True))
    # a transposed incoming gradient and an element offset that breaks the 16-byte alignment
    odd = torch.randn(3 * 40 * 256 + 1, device="cuda").to(torch.bfloat16)[1:].view(3, 40, 256)
    ra, za = gated_residual_norm(odd, one.repeat(3, 1, 1), v["y"], v["shift"], v["scale"])
    rb, zb = gated_residual_norm(odd.clone(), one.repeat(3, 1, 1), v["y"], v["shift"], v["scale"])
    assert torch.equal(ra, rb) and float((za.float() - zb.float()).abs().max()) <= 2 ** -8 * float(zb.float().abs().max())
    x4 = v["x"].clone().requires_grad_(True)
    _, z4 = gated_residual_norm(x4, one.repeat(3, 1, 1), v["y"], v["shift"], v["scale"], weight=v["weight"])
    dt = torch.autograd.grad(z4, x4, v["dz"].transpose(1, 2).contiguous().transpose(1, 2))[0]
    assert torch.equal(dt, dx2)


@pytest.mark.gpu
@pytest.mark.parametrize("b,t", [(0, 4), (2, 0)])
def test_no_tokens(b, t):
    from loractl_b200.block_ops import gated_residual_norm

    x = torch.zeros(b, t, 64, device="cuda", requires_grad=True)
    mods = [torch.ones(b, 1, 64, device="cuda", requires_grad=True) for _ in range(3)]
    w = torch.ones(64, device="cuda", requires_grad=True)
    r, z = gated_residual_norm(x, mods[0], x.detach(), mods[1], mods[2], weight=w)
    assert r.shape == z.shape == x.shape
    for g in torch.autograd.grad(z.sum() + r.sum(), mods + [w]):
        assert not g.any()


@pytest.mark.gpu
def test_zero_rows_nan_rows_and_determinism():
    """Padding rows (zeros) have finite gradients; a NaN row stays in its own row and in the sums over tokens; two
    runs are bit-identical."""
    from loractl_b200.block_ops import gated_residual_norm

    v = make(2, 900, 2048, torch.bfloat16, torch.bfloat16, seed=5)
    v["x"][:, 700:] = 0
    v["y"][:, 700:] = 0
    runs = []
    for _ in range(2):
        xs = [v[n].detach().requires_grad_(True) for n in ("x", "gate", "y", "shift", "scale", "weight")]
        out = gated_residual_norm(*xs[:5], weight=xs[5])
        runs.append([o.detach() for o in out] + list(torch.autograd.grad(out, xs, (v["dr"], v["dz"]))))
    assert all(torch.equal(p, q) and bool(torch.isfinite(p).all()) for p, q in zip(*runs))
    v["x"][1, 3, 5] = float("nan")
    r, z = gated_residual_norm(v["x"], v["gate"], v["y"], v["shift"], v["scale"])
    assert torch.isnan(z[1, 3]).all() and int(torch.isnan(z).any(-1).sum()) == 1 and int(torch.isnan(r).sum()) == 1


@pytest.mark.gpu
def test_captured_forward_and_backward_replay():
    """Forward and backward in a CUDA graph, replayed on new contents, with another stream's eager calls between."""
    from loractl_b200.block_ops import gated_residual_norm

    v = make(1, 200, 512, torch.bfloat16, torch.bfloat16, seed=6)
    names = ("x", "gate", "y", "shift", "scale")
    static = [v[n].detach().clone() for n in names]

    def step(src):
        xs = [s.detach().requires_grad_(True) for s in src]
        out = gated_residual_norm(*xs)
        return list(out) + list(torch.autograd.grad(out, xs, (v["dr"], v["dz"])))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    new = make(1, 200, 512, torch.bfloat16, torch.bfloat16, seed=7)
    for s, n in zip(static, names):
        s.copy_(new[n])
    graph.replay()
    with torch.cuda.stream(side):
        other = step([new[n] for n in names])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, other))


@pytest.mark.gpu
@pytest.mark.parametrize("h", [64, 65])
def test_rows_whose_squares_overflow(h):
    """A row above 1.8e19 has an infinite sum of squares in f32: it normalises to zero, as the f32 tensor ops have it, and
    touches no other row."""
    from loractl_b200.block_ops import modulated_zrmsnorm

    v = make(1, 5, h, torch.float32, torch.float32, seed=9)
    v["x"][0, 2] *= 1e25
    z = modulated_zrmsnorm(v["x"], v["weight"], v["shift"], v["scale"])
    x = v["x"]
    ref = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * (1 + v["weight"]) * (1 + v["scale"]) + v["shift"]
    assert torch.equal(z[0, 2], v["shift"][0, 0]) and torch.equal(ref[0, 2], z[0, 2])
    assert float((z - ref).abs().max()) <= 1e-5 * float(ref.abs().max())


@pytest.mark.gpu
def test_many_samples():
    """More samples than a grid's second axis has places, one token each: every sample's own sums, and the weight's over all."""
    from loractl_b200.block_ops import modulated_zrmsnorm

    b, h = 70_001, 8
    v = make(b, 1, h, torch.float32, torch.float32, seed=8)
    xs = [v[n].detach().requires_grad_(True) for n in ("x", "weight", "shift", "scale")]
    z = modulated_zrmsnorm(*xs)
    dx, dw, dshift, dscale = torch.autograd.grad(z, xs, v["dz"])
    ref = {n: v[n].detach().double().requires_grad_(True) for n in ("x", "weight", "shift", "scale")}
    _, rz = formula(ref, "zrms", False, 1.0, two=False)
    rdx, rdw, rdshift, rdscale = torch.autograd.grad(rz, [ref[n] for n in ("x", "weight", "shift", "scale")], v["dz"].double())
    close(z.detach(), rz.detach(), torch.float32, what="z")
    close(dx, rdx, torch.float32, rdx.abs().max() * 4, "x")
    assert torch.equal(dshift, v["dz"])
    close(dscale, rdscale, torch.float32, rdscale.abs().max(), "scale")
    c = v["x"].double()
    rh = (c / (c.square().mean(-1, keepdim=True) + EPS).sqrt()).abs()
    terms = (v["dz"].double().abs() * rh * (1 + v["scale"].detach().double()).abs()).sum((0, 1))
    close(dw, rdw, torch.float32, terms, "weight")


@pytest.mark.gpu
def test_differentiable_once():
    from loractl_b200.block_ops import gated_residual_norm

    v = make(1, 4, 64, torch.float32, torch.float32)
    x = v["x"].requires_grad_(True)
    _, z = gated_residual_norm(x, v["gate"], v["y"], v["shift"], v["scale"])
    (dx,) = torch.autograd.grad(z.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dx.sum().backward()
    _, z = gated_residual_norm(x, v["gate"], v["y"], v["shift"], v["scale"])
    z.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        z.sum().backward()
    _, z = gated_residual_norm(x, v["gate"], v["y"], v["shift"], v["scale"])
    v["y"].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()


@pytest.mark.gpu
def test_refusals():
    from loractl_b200 import _lib as L
    from loractl_b200.block_ops import gated_residual_norm, modulated_zrmsnorm

    v = make(2, 4, 64, torch.float32, torch.float32)
    args = [v[n] for n in ("x", "gate", "y", "shift", "scale")]
    with pytest.raises(ValueError, match="norm must be"):
        gated_residual_norm(*args, norm="batch")
    with pytest.raises(ValueError, match="gate and y are needed"):
        gated_residual_norm(args[0], args[1], None, *args[3:])
    with pytest.raises(ValueError, match="agree in shape and dtype"):
        gated_residual_norm(args[0], args[1], args[2].bfloat16(), *args[3:])
    with pytest.raises(ValueError, match="gate must be"):
        gated_residual_norm(args[0], args[1][:1], *args[2:])
    with pytest.raises(ValueError, match="weight must hold"):
        gated_residual_norm(*args, weight=torch.zeros(63, device="cuda"))
    with pytest.raises(TypeError, match="dtype"):
        gated_residual_norm(args[0].half(), args[1], args[2].half(), *args[3:])
    with pytest.raises(TypeError, match="dtype"):
        modulated_zrmsnorm(args[0], None, args[3].half(), args[4])
    with pytest.raises(RuntimeError, match="CUDA"):
        modulated_zrmsnorm(args[0].cpu(), None, args[3], args[4])
    with pytest.raises(RuntimeError, match="x on"):
        modulated_zrmsnorm(args[0], None, args[3].cpu(), args[4])
    wide = torch.zeros(1, 1, 16392, device="cuda")
    with pytest.raises(L.LqError, match="16384"):
        modulated_zrmsnorm(wide, None, wide, wide)


def test_library_refuses_bad_arguments_on_the_host():
    """The C entry's own checks, which come before any launch: no GPU is needed."""
    import ctypes as C

    from loractl_b200 import _lib as L

    a, g = L.ResidualNormArgs(), L.ResidualNormGrads()
    call = lambda: L.lib().lq_residual_norm_fwd(C.byref(a), None)
    assert L.lib().lq_residual_norm_fwd(None, None) == L.LQ_ERR_INVALID
    a.dtype = 7
    assert call() == L.LQ_ERR_INVALID and b"dtype" in L.lib().lq_last_error()
    a.dtype, a.samples, a.tokens, a.h = L.LQ_BF16, 1, 1, 16385
    assert call() == L.LQ_ERR_INVALID and b"16384" in L.lib().lq_last_error()
    a.h = 64
    assert call() == L.LQ_ERR_INVALID and b"NULL" in L.lib().lq_last_error()
    a.x = a.shift = a.scale = a.z = 16
    a.post_weight = 16
    assert call() == L.LQ_ERR_INVALID and b"y is NULL" in L.lib().lq_last_error()
    a.post_weight, a.y = None, 16
    assert call() == L.LQ_ERR_INVALID and b"gate" in L.lib().lq_last_error()
    a.y, a.samples, a.tokens = None, 1 << 20, 1 << 20
    assert call() == L.LQ_ERR_INVALID and b"2^31" in L.lib().lq_last_error()
    g.dgate = 16
    a.samples, a.tokens = 1, 1
    assert L.lib().lq_residual_norm_bwd(C.byref(a), C.byref(g), None, 0, None) == L.LQ_ERR_INVALID
    assert b"need y" in L.lib().lq_last_error()
    a.samples, a.tokens, a.x = 0, 5, None
    assert call() == L.LQ_OK
