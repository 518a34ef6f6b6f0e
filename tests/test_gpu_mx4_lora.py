"""An adapter on a microscaled weight as one call: values and all gradients against 64-bit formulas, the flat gradient
buffer, streams and captured graphs, and what is left to plain tensor ops.

Tolerances, with the factors rounded to bf16 on both sides.  Forward: the product's bound (tests/test_gpu_mx4.py); s * H is
rounded to bf16, so the delta is off by 2^-8 of sum |s H| |B|; y is rounded once or, for few tokens, the product and the
sum each, 2^-8 of either.  Backward: dH = s dY B^T is an f32 sum that is rounded to bf16 before dX and dA use it, s H
before dB does: 2^-8 of sum |dH| |A|, |X|^T |dH|, |s H|^T |dY|.  Reductions on the tensor cores step 16 products at a time,
each step 2^-22 of what has been added up: (len / 16 + 16) 2^-22 of the sum of magnitudes, the 16 for joined ranges; H's
and dH's own come in through the same sums of magnitudes.  1.02 covers the products of these small terms."""
import pytest
import torch

BF = torch.bfloat16
HALF = 2.0 ** -8


def steps(length):
    return (length / 16 + 16) * 2.0 ** -22


def site(n, m, k, r, seed=0, lead=(), bias=True):
    import loractl_b200 as lb

    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    lin = torch.nn.Linear(k, m, bias=bias).cuda()
    with torch.no_grad():
        lin.weight.copy_(rand(m, k) * 0.1)
    lora = lb.LoraLinear(lb.Mx4Linear.from_linear(lin), r, 2.0 * r, device="cuda")
    with torch.no_grad():
        lora.delta.lora_a.copy_(rand(k, r) * k ** -0.5)
        lora.delta.lora_b.copy_(rand(r, m) * 0.3)
    x = rand(*lead, n, k).to(BF).requires_grad_(True)
    dy = rand(*lead, n, m).to(BF)
    return lin, lora, x, dy


def check(lin, lora, x, dy, y, dx, da, db):
    import loractl_b200 as lb

    layer, d = lora.base.inner, lora.delta
    m, k = layer.weight.shape
    s = d.scaling
    a, b = d.lora_a.detach().to(BF).double(), d.lora_b.detach().to(BF).double()
    w = layer.weight.dequantize().double()
    xs, dys = x.detach().double().reshape(-1, k), dy.double().reshape(-1, m)
    xq = lb.mx4_quantize(x).dequantize().double()
    h, hm = s * (xs @ a), abs(s) * (xs.abs() @ a.abs())
    base = xq @ w.t() + (0.0 if lin.bias is None else lin.bias.double())
    ref = base + h @ b
    lim = HALF * (base.abs() + ref.abs() + h.abs() @ b.abs()) + (2 * k / 64 + 8) * 2.0 ** -23 * (xq.abs() @ w.abs().t())
    lim += steps(k + d.rank) * (hm @ b.abs()) + 2.0 ** -23 * base.abs()
    refs = {"y": (y, ref, lim)}
    dh, dhm = s * (dys @ b.t()), abs(s) * (dys.abs() @ b.t().abs())
    if dx is not None:
        mag = dys.abs() @ w.abs()
        ref = dys @ w + dh @ a.t()
        refs["dx"] = (dx, ref, HALF * (ref.abs() + dh.abs() @ a.t().abs()) + steps(m) * (mag + 2 * (dhm @ a.t().abs())))
    n = xs.shape[0]
    refs["da"] = (da, xs.t() @ dh, HALF * (xs.t().abs() @ dh.abs()) + (steps(m) + steps(n)) * (xs.t().abs() @ dhm))
    refs["db"] = (db, h.t() @ dys, HALF * (h.t().abs() @ dys.abs()) + (steps(k) + steps(n)) * (hm.t() @ dys.abs()))
    for name, (got, ref, lim) in refs.items():
        err = (got.detach().double().reshape(ref.shape) - ref).abs()
        assert bool((err <= 1.02 * lim).all()), (name, float((err / lim.clamp(min=1e-300)).max()))
    lb.check_device_status()


# few tokens and outputs (a kernel of its own adds the delta), then pairs of SMs (two to five k-blocks, ragged edges);
# backward below 256 tokens, at an input of at most 192 and above; ranks of one to four k-blocks
SITES = [(1, 8, 32, 1), (33, 4104, 512, 4), (1, 6152, 64, 100), (5, 304, 96, 4), (33, 72, 1184, 2), (77, 512, 288, 16), (129, 520, 64, 3), (256, 512, 512, 16), (300, 1000, 160, 8),
         (301, 64, 1024, 64), (1000, 8, 224, 5), (2000, 2048, 288, 16), (1801, 1928, 544, 72), (2050, 1544, 32, 256), (1793, 2056, 1312, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,m,k,r", SITES)
def test_values_and_gradients_match_64_bits(n, m, k, r):
    lin, lora, x, dy = site(n, m, k, r, seed=n)
    y = lora(x)
    assert y.dtype == BF and y.shape == (n, m) and y.grad_fn.name() == "Mx4LoraBackward"
    dx, da, db = torch.autograd.grad(y, [x, lora.delta.lora_a, lora.delta.lora_b], dy)
    assert dx.shape == x.shape and dx.dtype == BF and da.dtype == db.dtype == torch.float32
    check(lin, lora, x, dy, y, dx, da, db)
    with torch.no_grad():
        assert torch.equal(lora(x), y)


@pytest.mark.gpu
@pytest.mark.parametrize("r", [1, 16, 100])
def test_every_place_of_the_delta(r):
    """A zero weight and one non-zero entry per row of x, A and B: each output is one known product, exact in bf16."""
    import loractl_b200 as lb

    for n, m, k in ((40, 136, 256), (2100, 1800, 256)):
        lora = lb.LoraLinear(lb.Mx4Linear(lb.mx4_quantize(torch.zeros(m, k, device="cuda"))), r, 1.0 * r, device="cuda")
        i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
        x, a, b = torch.zeros(n, k, device="cuda", dtype=BF), torch.zeros(k, r, device="cuda"), torch.zeros(r, m, device="cuda")
        x[i, (i * 37) % k] = torch.exp2((i % 11 - 5).float()).to(BF)
        a[torch.arange(k, device="cuda"), (torch.arange(k, device="cuda") * 7) % r] = 2.0
        b[(j * 5) % r, j] = torch.exp2((j % 7 - 3).float())
        with torch.no_grad():
            lora.delta.lora_a.copy_(a), lora.delta.lora_b.copy_(b)
        assert torch.equal(lora(x).double(), x.double() @ a.double() @ b.double())


@pytest.mark.gpu
def test_leading_axes_strides_and_no_tokens():
    lin, lora, x, dy = site(9, 64, 96, 4, lead=(3, 2))
    wide = torch.randn(3, 2, 9, 101, device="cuda").to(BF)
    xs = wide[..., 5:].detach().requires_grad_(True)  # strided rows that start off 16 bytes
    dys = dy.transpose(0, 1).contiguous().transpose(0, 1)
    y = lora(xs)
    grads = torch.autograd.grad(y, [xs, lora.delta.lora_a, lora.delta.lora_b], dys)
    assert y.shape == (3, 2, 9, 64) and grads[0].shape == xs.shape
    check(lin, lora, xs, dys, y, *grads)
    none = x[:, :, :0].detach().requires_grad_(True)
    y = lora(none)
    grads = torch.autograd.grad(y, [none, lora.delta.lora_a, lora.delta.lora_b], torch.zeros_like(y))
    assert y.shape == (3, 2, 0, 64) and grads[0].shape == none.shape and not grads[1].any() and not grads[2].any()


@pytest.mark.gpu
def test_only_what_is_asked_for():
    """Frozen x (the first block's), frozen factors, no bias."""
    lin, lora, x, dy = site(40, 64, 96, 4, bias=False)
    full = torch.autograd.grad(lora(x), [x, lora.delta.lora_a, lora.delta.lora_b], dy)
    check(lin, lora, x, dy, lora(x), *full)
    part = torch.autograd.grad(lora(x.detach()), [lora.delta.lora_a, lora.delta.lora_b], dy)
    assert torch.equal(part[0], full[1]) and torch.equal(part[1], full[2])
    for p in (lora.delta.lora_a, lora.delta.lora_b):
        p.requires_grad_(False)
    assert torch.equal(torch.autograd.grad(lora(x), x, dy)[0], full[0])
    assert not lora(x.detach()).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 300])
def test_gradients_add_into_the_flat_buffer(n):
    import loractl_b200 as lb

    lin, lora, x, dy = site(n, 64, 224, 4)
    d = lora.delta
    want = torch.autograd.grad(lora(x), [d.lora_a, d.lora_b], dy)
    flat = lb.FlatAdapters(lb.LoraAdapters([d], ["site"]), "cuda")
    flat.zero_grad()
    for times in (1, 2):  # twice: accumulated
        lora(x).backward(dy)
        for i, p in enumerate((d.lora_a, d.lora_b)):
            assert p.grad.data_ptr() == flat.grad_views(0)[i].data_ptr()
            assert bool(((p.grad - times * want[i]).abs() <= 2.0 ** -23 * times * want[i].abs()).all())
    d.lora_a.grad = d.lora_b.grad = None  # the caller wants autograd's own
    lora(x).backward(dy)
    assert torch.equal(d.lora_a.grad, want[0]) and torch.equal(d.lora_b.grad, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("n,m", [(40, 136), (2000, 2048)])
def test_streams_capture_determinism_and_new_factors(n, m):
    lin, lora, x, dy = site(n, m, 288, 8)
    d = lora.delta
    wrt = [x, d.lora_a, d.lora_b]
    run = lambda: (lambda y: [y.detach(), *torch.autograd.grad(y, wrt, dy)])(lora(x))
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(4):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            outs.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))
    del outs
    graphs, res = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res.append(run())
        graphs.append(g)
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = run()
    assert all(torch.equal(a, b) for o in res for a, b in zip(o, want))
    with torch.no_grad():
        d.lora_b.mul_(-1.0)  # the bf16 operands follow the factors
    y = lora(x)
    grads = torch.autograd.grad(y, wrt, dy)
    check(lin, lora, x, dy, y, *grads)


@pytest.mark.gpu
def test_nan_and_inf_stay_in_their_rows():
    for n, m in ((40, 136), (2000, 2048)):
        _, lora, x, _ = site(n, m, 288, 8)
        good = lora(x.detach())
        bad = x.detach().clone()
        bad[3, 7], bad[5, 40] = float("nan"), float("inf")
        y = lora(bad)
        rows = torch.zeros(n, dtype=torch.bool, device="cuda")
        rows[3] = rows[5] = True
        assert bool(torch.isnan(y[rows]).all()) and torch.equal(y[~rows], good[~rows])


@pytest.mark.gpu
def test_differentiable_once_retained_and_changed_in_place():
    _, lora, x, dy = site(20, 64, 96, 4)
    y = lora(x)
    g = torch.autograd.grad(y, x, dy, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.float().sum().backward()
    first = torch.autograd.grad(y, x, dy, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], first)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, x, dy)
    y = lora(x)
    with torch.no_grad():
        lora.delta.lora_a.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, x, dy)


@pytest.mark.gpu
def test_what_plain_ops_keep():
    """f32 activations, widths off 8 and dropout: the delta in plain tensor ops, as before."""
    import loractl_b200 as lb

    _, lora, x, _ = site(20, 64, 96, 4)
    layer, d = lora.base.inner, lora.delta
    xf = x.detach().float()
    assert torch.equal(lora(xf), layer(xf) + d(xf))
    _, odd, xo, _ = site(20, 63, 96, 4)
    assert torch.equal(odd(xo), odd.base.inner(xo) + odd.delta(xo))
    drop = lb.LoraLinear(layer, 4, 8.0, dropout_prob=0.5, device="cuda")
    with torch.no_grad():
        drop.delta.lora_b.normal_()
    assert not torch.equal(drop(x), drop(x))
    drop.eval()
    assert torch.equal(drop(x), drop(x)) and drop(x).grad_fn.name() == "Mx4LoraBackward"


@pytest.mark.gpu
def test_refusals():
    from loractl_b200 import _lib as L

    _, lora, x, _ = site(20, 64, 96, 4)
    w, d = lora.base.inner.weight, lora.delta
    call = lambda x=x, a=d.lora_a, b=d.lora_b, mirror=d.operand_mirror(), m=64: L.ext().mx4_lora_linear(
        x, w.codes, w.scales, m, 96, None, a, b, 1.0, mirror, None, None)
    call()
    with pytest.raises(TypeError, match="bf16"):
        call(x=x.float())
    with pytest.raises(ValueError, match="d_in"):
        call(x=x[:, :64])
    with pytest.raises(RuntimeError, match="lora_a is on cpu"):
        call(a=d.lora_a.cpu())
    with pytest.raises(ValueError, match="lora_a must be"):
        call(b=d.lora_b.t())
    with pytest.raises(ValueError, match="mirror is too small"):
        call(mirror=d.operand_mirror()[:256])
    with pytest.raises(ValueError, match="d_in"):
        lora(torch.randn(3, 64, device="cuda").to(BF))


def test_library_refuses_bad_arguments_on_the_host():
    """Bad sizes and pointers end as codes before anything touches a device."""
    from loractl_b200 import _lib as L

    lib, p = L.lib(), 1 << 20
    fwd = lambda n=4, m=64, k=96, r=4, mirror=p, x=p, y=p, ws=p, size=1 << 40, codes=p: lib.lq_mx4_lora_fwd(
        x, n, codes, p, m, k, None, mirror, r, 1.0, y, None, ws, size, None)
    bwd = lambda n=4, m=64, k=96, r=4, mirror=p, x=p, dy=p, dx=p: lib.lq_mx4_lora_bwd(dy, x, None, n, p, p, m, k, mirror, r, 1.0, dx, None, None, 0,
                                                                                     None, 0, None)
    for bad in (dict(n=-1), dict(m=60), dict(m=0), dict(k=100), dict(k=0), dict(r=0), dict(r=257), dict(mirror=None), dict(mirror=p + 64),
                dict(x=None), dict(x=p + 8)):
        assert fwd(**bad) == L.LQ_ERR_INVALID and lib.lq_last_error()
        assert bwd(**bad) == L.LQ_ERR_INVALID and lib.lq_last_error()
    for bad in (dict(y=None), dict(y=p + 2), dict(ws=None), dict(ws=p + 16), dict(codes=None)):
        assert fwd(**bad) == L.LQ_ERR_INVALID
    for bad in (dict(dy=None), dict(dy=p + 2), dict(dx=p + 8)):
        assert bwd(**bad) == L.LQ_ERR_INVALID
    assert fwd(size=64) == L.LQ_ERR_WORKSPACE
    assert fwd(n=0) == 0
    for n, m, k, r in ((0, 64, 96, 4), (4, 64, 96, 0), (4, 64, 96, 257)):
        assert lib.lq_mx4_lora_workspace_bytes(n, m, k, r, 0) == 0 == lib.lq_mx4_lora_workspace_bytes(n, m, k, r, 1)
