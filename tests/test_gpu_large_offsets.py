"""Tensors of more than 2^31 elements through the step's operators: the last rows of a large call equal, bit for bit, a call
on those rows alone (every row is computed on its own), and a norm over them is the norm."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_residual_norm():
    from loractl_b200.block_ops import gated_residual_norm

    t, h, tail = 350_003, 6144, 5
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(1, t, h, dtype=torch.bfloat16, device="cuda").normal_(generator=g).requires_grad_(True)
    y = torch.empty(1, t, h, dtype=torch.bfloat16, device="cuda").normal_(generator=g).requires_grad_(True)
    mods = [torch.randn(1, 1, h, generator=g, device="cuda").bfloat16() for _ in range(3)]
    assert x.numel() > 2 ** 31
    r, z = gated_residual_norm(x, mods[0], y, mods[1], mods[2])
    dx, dy = torch.autograd.grad((r, z), (x, y), (x.detach(), y.detach()))
    xs, ys = (v.detach()[:, -tail:].clone().requires_grad_(True) for v in (x, y))
    rs, zs = gated_residual_norm(xs, mods[0], ys, mods[1], mods[2])
    dxs, dys = torch.autograd.grad((rs, zs), (xs, ys), (xs.detach(), ys.detach()))
    for big, small in ((r, rs), (z, zs), (dx, dxs), (dy, dys)):
        assert torch.equal(big[:, -tail:], small)


def test_quantise_and_back():
    import loractl_b200 as lb

    n, k, tail = 33_001, 65_536, 7
    x = torch.empty(n, k, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    assert x.numel() > 2 ** 31
    big, small = lb.mx4_quantize(x).dequantize(torch.bfloat16), lb.mx4_quantize(x[-tail:]).dequantize(torch.bfloat16)
    assert torch.equal(big[-tail:], small)


@pytest.mark.parametrize("n,m", [(70_001, 32_768), (100, 22_000_000)])
def test_product(n, m):
    """More than 2^31 outputs, by the pairs' kernel and by the stream's."""
    import loractl_b200 as lb

    g = torch.Generator(device="cuda").manual_seed(2)
    x, w = (torch.randn(v, 64, generator=g, device="cuda").bfloat16() for v in (n, m))
    y = lb.mx4_matmul_t(lb.mx4_quantize(x), lb.mx4_quantize(w))
    assert y.numel() > 2 ** 31
    xd, wd = (lb.mx4_quantize(v).dequantize() for v in (x[-3:], w[-5:]))
    ref = xd.double() @ wd.double().t()
    tail = y[-3:, -5:].double()
    assert bool(((tail - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-5 * (xd.abs() @ wd.abs().t())).all())
    lb.check_device_status()


@pytest.mark.parametrize("n,m", [(70_001, 32_768), (100, 22_000_000)])
def test_adapter(n, m):
    """The same with an adapter, and for the first its gradients: bounds as in tests/test_gpu_mx4_lora.py, for a corner."""
    import loractl_b200 as lb

    k, r, half = 64, 4, 2.0 ** -8
    steps = lambda length: (length / 16 + 16) * 2.0 ** -22
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(n, k, generator=g, device="cuda").bfloat16().requires_grad_(True)
    layer = lb.Mx4Linear(lb.mx4_quantize(torch.randn(m, k, generator=g, device="cuda").bfloat16()))
    lora = lb.LoraLinear(layer, r, 2.0 * r, device="cuda")
    d = lora.delta
    with torch.no_grad():
        d.lora_a.normal_(generator=g), d.lora_b.normal_(generator=g)
    y = lora(x)
    assert y.numel() > 2 ** 31
    a, b = d.lora_a.detach().bfloat16().double(), d.lora_b.detach().bfloat16().double()
    few = layer.weight.dequantize(torch.bfloat16)[-5:].double()
    xs, xq = x.detach()[-3:].double(), lb.mx4_quantize(x[-3:]).dequantize().double()
    base, h = xq @ few.t(), 2.0 * (xs @ a)
    ref = base + h @ b[:, -5:]
    lim = half * (base.abs() + ref.abs() + h.abs() @ b[:, -5:].abs()) + steps(k) * (xq.abs() @ few.abs().t() + 2 * (xs.abs() @ a.abs()) @ b[:, -5:].abs())
    assert bool(((y.detach()[-3:, -5:].double() - ref).abs() <= 1.02 * lim).all())
    if n > m:
        dy = torch.empty(n, m, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
        dx, db = torch.autograd.grad(y, [x, d.lora_b], dy)
        w, dys = layer.weight.dequantize().double(), dy[-3:].double()
        dh, dhm = 2.0 * (dys @ b.t()), 2.0 * (dys.abs() @ b.t().abs())
        ref = dys @ w + dh @ a.t()
        lim = half * (ref.abs() + dh.abs() @ a.t().abs()) + steps(m) * (dys.abs() @ w.abs() + 2 * (dhm @ a.t().abs()))
        assert bool(((dx[-3:].double() - ref).abs() <= 1.02 * lim).all())
        h, hm, last = 2.0 * (x.detach().double() @ a), 2.0 * (x.detach().double().abs() @ a.abs()), dy[:, -5:].double()
        lim = half * (h.abs().t() @ last.abs()) + (steps(k) + steps(n)) * (hm.t() @ last.abs())
        assert bool(((db[:, -5:].double() - h.t() @ last).abs() <= 1.02 * lim).all())
    lb.check_device_status()


def test_gradient_norm():
    import loractl_b200 as lb

    n = 2 ** 31 + 77
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    g[-1] = 4096.0
    want = (0.25 * (n - 1) + 4096.0 ** 2) ** 0.5
    assert abs(float(lb.clip_grad_norm([g], want / 2)) - want) <= 2 ** -23 * want
    assert float(g[-1]) == 2048.0 and float(g[-2]) == 0.25
