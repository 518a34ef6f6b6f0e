"""Microscaled 4-bit floats: quantisation against the definition element by element (exact), the product and the
gradient against 64-bit products of the dequantised operands, the layer in the places that take one, and the refusals.

Tolerances.  Quantisation is exact arithmetic and one rounding: equal.  Products of two elements and their scales are
exact; the tensor core adds 64 of them at a time onto an f32 accumulator, and each such step may round (or cut) the
sum twice by 2^-23 of what has been added up, so (2 k / 64 + 8) 2^-23 of sum |x w| bounds the f32 result, joined ranges
included; a bf16 output adds half a step, 2^-8 of its value.  The bf16 gradient's reduction runs over d_out in steps
of 16 with the same reasoning; the f32 gradient has the bound of adding one product at a time, d_out 2^-24 of sum |dy w|."""
import pytest
import torch

BF, F = torch.bfloat16, torch.float32
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def definition(x):
    """(codes, scale bytes, values) of x [rows, k] in 64 bits on the CPU, by distance to the grid."""
    x = x.detach().double().cpu()
    rows, k = x.shape
    v = x.reshape(rows, k // 32, 32)
    top = v.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.where((top > 0) & torch.isfinite(top), top, torch.ones_like(top))))
    e = torch.where(torch.exp2(e) > top, e - 1, e)  # log2 may round up to a power of two not reached
    e = torch.where(top > 0, e - 2, torch.full_like(e, -127.0)).clamp(-127, 125)
    a = v.abs() / torch.exp2(e)
    dist = (a.clamp(max=6.0).unsqueeze(-1) - GRID).abs()
    dist = torch.where(torch.isnan(dist), torch.zeros_like(dist), dist)
    best = dist.amin(-1, keepdim=True)
    near = dist == best
    code = torch.where(near, torch.arange(8), 99).amin(-1)
    high = torch.where(near, torch.arange(8), -1).amax(-1)
    code = torch.where((high != code) & (code % 2 == 1), high, code)  # a tie goes to the even code
    bad = ~torch.isfinite(top)
    value = torch.copysign(GRID[code], v) * torch.exp2(e)
    value = torch.where(bad, torch.full_like(value, float("nan")), value)
    scale = torch.where(bad, torch.full_like(e, 128.0), e) + 127
    sign = torch.signbit(v).long() * 8
    return (code + sign).reshape(rows, k), scale.squeeze(-1).long(), value.reshape(rows, k)


def sample(rows, k, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device="cuda") * 3
    x *= 10.0 ** torch.randint(-6, 4, (rows, k // 32, 1), generator=g, device="cuda").float().expand(rows, k // 32, 32).reshape(rows, k)
    x[torch.rand(rows, k, generator=g, device="cuda") < 0.05] = 0
    return x.to(dtype)


def special_rows(dtype):
    """Ties and their neighbours, whole blocks of zeros, subnormals, the largest values, Inf and NaN."""
    rows = []
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.75, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0])
    for p in (-120, -30, 0, 30, 100):
        rows.append(torch.cat([ties, -ties]) * 2.0 ** p)
    step = 2.0 ** -7 if dtype == BF else 2.0 ** -20
    rows += [torch.cat([ties * (1 + step), -ties * (1 - step)]), torch.zeros(32), -torch.zeros(32)]
    rows.append(torch.full((32,), 1e-40))
    rows.append(torch.cat([torch.full((31,), 2.0 ** -126), torch.tensor([2.0 ** -133])]))
    rows.append(torch.full((32,), float(torch.finfo(dtype).max)))
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.randn(32)
        r[17] = bad
        rows.append(r)
    return torch.stack(rows).to(dtype).cuda()


def check_quantised(q, x):
    codes, scales, values = definition(x)
    got_codes, got_scales = (t.cpu().long() for t in q.unpack())
    assert torch.equal(got_scales, scales)
    fine = (scales != 255).repeat_interleave(32, dim=1)
    assert torch.equal(got_codes[fine], codes[fine])
    for dtype in (F, BF):
        out = q.dequantize(dtype).double().cpu()
        assert torch.equal(torch.isnan(out), torch.isnan(values)) and torch.equal(out[fine], values[fine])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (33, 256), (128, 288), (129, 512), (257, 32), (300, 1184), (1, 6144)])
@pytest.mark.parametrize("dtype", [F, BF])
def test_quantise_is_the_definition(rows, k, dtype):
    import loractl_b200 as lb

    x = sample(rows, k, dtype)
    check_quantised(lb.mx4_quantize(x), x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, BF])
def test_quantise_borders(dtype):
    import loractl_b200 as lb

    x = special_rows(dtype)
    check_quantised(lb.mx4_quantize(x), x)


@pytest.mark.gpu
def test_quantise_strides_and_empty():
    import loractl_b200 as lb

    x = sample(64, 512, BF, seed=1)
    q = lb.mx4_quantize(x)
    same = lambda a, b: torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    wide = torch.zeros(64, 1000, dtype=BF, device="cuda")
    for off in (0, 8, 3):  # rows of a wider tensor, on 16 bytes and off them
        wide[:, off:off + 512] = x
        assert same(lb.mx4_quantize(wide[:, off:off + 512]), q)
    assert same(lb.mx4_quantize(x.t().contiguous().t()), q) and same(lb.mx4_quantize(x.view(4, 16, 512)), q)
    assert same(lb.mx4_quantize(x[:1].expand(64, 512)), lb.mx4_quantize(x[:1].repeat(64, 1)))
    e = lb.mx4_quantize(x[:0])
    assert e.shape == (0, 512) and e.dequantize().shape == (0, 512) and e.unpack()[1].shape == (0, 16)
    assert lb.mx4_matmul_t(e, q).shape == (0, 64) and lb.mx4_matmul_t(q, e).shape == (64, 0)


def bound(x, w, k, dtype, ref):
    mag = x.abs() @ w.abs().t()
    return (2 * k / 64 + 8) * 2.0 ** -23 * mag + (2.0 ** -8 if dtype == BF else 2.0 ** -24) * ref.abs()


PRODUCTS = [(1, 1, 32), (1, 128, 256), (2, 130, 288), (16, 300, 512), (17, 64, 96), (33, 1000, 1184), (64, 128, 2048), (77, 515, 2592), (128, 256, 320),
            (129, 129, 64), (200, 40, 512), (255, 769, 544), (256, 256, 256), (300, 2000, 1024), (513, 1000, 6144), (1, 6144, 16384), (1000, 7, 160)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,m,k", PRODUCTS)
@pytest.mark.parametrize("dtype", [BF, F])
def test_product_matches_64_bits(n, m, k, dtype):
    import loractl_b200 as lb

    g = torch.Generator(device="cuda").manual_seed(n + m)
    x = torch.randn(n, k, generator=g, device="cuda") * torch.exp(torch.randn(n, 1, generator=g, device="cuda"))
    w = torch.randn(m, k, generator=g, device="cuda") * torch.exp2(torch.randint(-8, 8, (m, 1), generator=g, device="cuda").float())
    bias = torch.randn(m, generator=g, device="cuda")
    xq, wq = lb.mx4_quantize(x), lb.mx4_quantize(w)
    xd, wd = xq.dequantize().double(), wq.dequantize().double()
    for b in (None, bias):
        y = lb.mx4_matmul_t(xq, wq, b, dtype)
        ref = xd @ wd.t() + (0.0 if b is None else b.double())
        assert y.shape == (n, m) and y.dtype == dtype
        err = (y.double() - ref).abs()
        lim = bound(xd, wd, k, dtype, ref) + (0.0 if b is None else 2.0 ** -23 * b.double().abs())
        assert bool((err <= lim).all()), float((err / lim.clamp(min=1e-300)).max())
    lb.check_device_status()


@pytest.mark.gpu
def test_product_of_units_finds_every_place():
    """One non-zero element per row: each output is one known product, so a wrong row, column, scale or k shows."""
    import loractl_b200 as lb

    n, m, k = 200, 333, 1056
    x, w = torch.zeros(n, k, device="cuda"), torch.zeros(m, k, device="cuda")
    i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    x[i, (i * 37) % k] = torch.exp2((i % 23 - 11).float())
    w[j] = torch.exp2(((j.unsqueeze(1) * 5 + torch.arange(k, device="cuda") // 32) % 19 - 9).float())
    ref = x.double() @ w.double().t()
    for rows in (1, 20, 100, n):
        y = lb.mx4_matmul_t(lb.mx4_quantize(x[:rows]), lb.mx4_quantize(w), dtype=F)
        assert torch.equal(y.double(), ref[:rows])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 100, 300])
def test_nan_blocks_reach_their_rows_only(n):
    import loractl_b200 as lb

    x, w = sample(n, 512, BF, seed=2), sample(300, 512, BF, seed=3)
    good = lb.mx4_matmul_t(lb.mx4_quantize(x), lb.mx4_quantize(w))
    x[1, 40], w[200, 500] = float("inf"), float("nan")
    y = lb.mx4_matmul_t(lb.mx4_quantize(x), lb.mx4_quantize(w))
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1], bad[:, 200] = True, True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], good[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("n,m,k", [(1, 8, 32), (5, 300, 96), (77, 515, 288), (256, 512, 512), (300, 1001, 1024), (1, 1, 64)])
@pytest.mark.parametrize("dtype", [BF, F])
def test_layer_and_gradient(n, m, k, dtype):
    import loractl_b200 as lb

    g = torch.Generator(device="cuda").manual_seed(n * m)
    lin = torch.nn.Linear(k, m).cuda()
    layer = lb.Mx4Linear.from_linear(lin)
    x = torch.randn(2, n, k, generator=g, device="cuda").to(dtype).requires_grad_(True)
    dy = torch.randn(2, n, m, generator=g, device="cuda").to(dtype)
    y = layer(x)
    dx = torch.autograd.grad(y, x, dy)[0]
    w = layer.weight.dequantize().double()
    xd = lb.mx4_quantize(x).dequantize().double()
    ref = xd @ w.t() + lin.bias.double()
    assert y.shape == (2, n, m) and y.dtype == dtype and dx.shape == x.shape and dx.dtype == dtype
    lim = bound(xd, w, k, dtype, ref) + 2.0 ** -23 * lin.bias.double().abs()
    assert bool(((y.detach().double().view(-1, m) - ref).abs() <= lim).all())
    d = dy.double().view(-1, m)
    ref, mag = d @ w, d.abs() @ w.abs()
    lim = ((2 * m / 16 + 8) * 2.0 ** -23 * mag + 2.0 ** -8 * ref.abs()) if dtype == BF else (m + 4) * 2.0 ** -24 * mag
    assert bool(((dx.double().view(-1, k) - ref).abs() <= lim).all())
    lb.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("n,m,k", [(1, 4104, 512), (3, 5000, 96), (130, 2056, 1024), (64, 8192, 32), (600, 6152, 512), (2600, 6152, 2048)])
@pytest.mark.parametrize("dtype", [BF, F])
def test_gradient_over_many_outputs(n, m, k, dtype):
    """Reductions that are cut into ranges: few rows, few columns, a last round of pairs."""
    import loractl_b200 as lb

    g = torch.Generator(device="cuda").manual_seed(n + m)
    w = lb.mx4_quantize(torch.randn(m, k, generator=g, device="cuda"))
    dy = (torch.randn(n, m, generator=g, device="cuda") * torch.exp(torch.randn(n, 1, generator=g, device="cuda"))).to(dtype)
    dx = lb.mx4_matmul_dx(dy, w)
    wd, d = w.dequantize().double(), dy.double()
    ref, mag = d @ wd, d.abs() @ wd.abs()
    lim = ((2 * m / 16 + 8) * 2.0 ** -23 * mag + 2.0 ** -8 * ref.abs()) if dtype == BF else (m + 4) * 2.0 ** -24 * mag
    assert dx.dtype == dtype and bool(((dx.double() - ref).abs() <= lim).all())
    assert torch.equal(lb.mx4_matmul_dx(dy, w), dx)
    lb.check_device_status()


@pytest.mark.gpu
def test_two_streams_capture_and_determinism():
    """Two products at once on two streams with their own workspaces, two captured graphs replayed in turn."""
    import loractl_b200 as lb

    x, w = sample(40, 4096, BF, seed=5), sample(700, 4096, BF, seed=6)
    layer = lb.Mx4Linear(lb.mx4_quantize(w))
    want = layer(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            outs.append(layer(x))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs, static, res = [], x.clone(), []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            xs = static.detach().requires_grad_(True)
            y = layer(xs)
            res.append((y, torch.autograd.grad(y, xs, torch.ones_like(y))[0]))
        graphs.append(g)
    static.copy_(sample(40, 4096, BF, seed=7))
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][0], layer(static)) and torch.equal(res[0][1], res[1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40, 300])
def test_operands_of_the_launch_before(n):
    """A product right behind the quantisation of its weight, and a linear right behind it, read what that wrote: the
    product's launch may start early, its reads may not."""
    import loractl_b200 as lb

    x = sample(n, 4096, BF, seed=8)
    xq = lb.mx4_quantize(x)
    for seed in range(4):
        w = sample(6000, 4096, BF, seed=10 + seed)
        lb.mx4_quantize(sample(6000, 4096, BF, seed=20 + seed))  # leaves other codes where the next allocation may lie
        torch.cuda.synchronize()
        wq = lb.mx4_quantize(w)
        y = lb.mx4_matmul_t(xq, wq)
        wq2 = lb.mx4_quantize(w)
        z = lb.Mx4Linear(wq2)(x)
        torch.cuda.synchronize()
        want = lb.mx4_matmul_t(xq, wq)
        assert torch.equal(y, want) and torch.equal(z, want)


@pytest.mark.gpu
def test_f32_gradient_over_the_whole_range():
    """dy from the smallest normal numbers to the largest, cut into three bf16 terms without overflow; Inf and NaN stay in
    their rows."""
    import loractl_b200 as lb

    w = lb.mx4_quantize(sample(96, 64, F, seed=30).clamp(-1, 1) * 2.0 ** -8)
    dy = torch.randn(6, 96, device="cuda")
    dy[0] *= 1e30
    dy[1, ::2], dy[1, 1::2] = 3.4e38, -3.3e38
    dy[2] *= 1e-30
    dy[3, 5], dy[4, 7] = float("inf"), float("nan")
    dx = lb.mx4_matmul_dx(dy, w)
    wd = w.dequantize().double()
    ref, mag = dy.double() @ wd, dy.double().abs() @ wd.abs()
    ok = [0, 1, 2, 5]
    assert bool(((dx.double() - ref)[ok].abs() <= 100 * 2.0 ** -24 * mag[ok]).all())
    assert torch.equal(torch.isnan(dx[4]), torch.isnan(ref[4])) and not torch.isfinite(dx[3]).any()


@pytest.mark.gpu
def test_layer_is_differentiable_once():
    import loractl_b200 as lb

    x = torch.randn(3, 64, device="cuda", requires_grad=True)
    layer = lb.Mx4Linear(lb.mx4_quantize(torch.randn(32, 64, device="cuda")))
    (dx,) = torch.autograd.grad(layer(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dx.sum().backward()


FIRST_CALL_CAPTURED = """
import torch
import loractl_b200 as lb
from loractl_b200.block_ops import gated_residual_norm
torch.manual_seed(0)
x = torch.randn(2, 8, 256, device="cuda")
mods = [torch.randn(2, 1, 256, device="cuda") for _ in range(3)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    r, z = gated_residual_norm(x, mods[0], x, mods[1], mods[2])
    y = lb.Mx4Linear(lb.mx4_quantize(z[0]))(z)
    norm = lb.clip_grad_norm([y, r], 1.0)
graph.replay()
torch.cuda.synchronize()
r2, z2 = gated_residual_norm(x, mods[0], x, mods[1], mods[2])
y2 = lb.Mx4Linear(lb.mx4_quantize(z2[0]))(z2)
norm2 = lb.clip_grad_norm([y2, r2], 1.0)
assert torch.equal(z, z2) and torch.equal(y, y2) and torch.equal(r, r2) and torch.equal(norm, norm2)
lb.check_device_status()
print("same")
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_may_be_captured():
    import subprocess
    import sys

    from tests.conftest import ROOT

    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout[-1000:] + r.stderr[-2000:]


CAPTURE_BESIDE_EAGER = """
import torch
import loractl_b200 as lb
from loractl_b200.block_ops import gated_residual_norm
x = torch.randn(2, 8, 64, device="cuda", requires_grad=True)
mods = [torch.randn(2, 1, 64, device="cuda", requires_grad=True) for _ in range(3)]
layer = lb.Mx4Linear(lb.mx4_quantize(torch.randn(32, 64, device="cuda")))
for op in (lambda: gated_residual_norm(x, mods[0], x, mods[1], mods[2])[1], lambda: layer(x)):
    living = op()
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            op().sum().backward()
    except RuntimeError as e:
        assert "capture" in str(e), e
    torch.cuda.synchronize()
    assert torch.isfinite(op()).all() and torch.isfinite(torch.autograd.grad(living.sum(), x)[0]).all()
print("usable")
"""


@pytest.mark.gpu
def test_capture_beside_a_living_eager_graph_ends_in_an_error():
    """A backward pass captured while an eager graph of the same leaves lives is torch's error about the capture, as with
    torch's own operators: the process, the context and the eager graph stay usable."""
    import subprocess
    import sys

    from tests.conftest import ROOT

    r = subprocess.run([sys.executable, "-c", CAPTURE_BESIDE_EAGER], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "usable" in r.stdout, r.stdout[-1000:] + r.stderr[-2000:]


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    import loractl_b200 as lb

    x = torch.zeros(4, 64, device="cuda")
    q = lb.mx4_quantize(x)
    with pytest.raises(ValueError, match="multiple of 32"):
        lb.mx4_quantize(torch.zeros(4, 48, device="cuda"))
    with pytest.raises(ValueError, match="multiple of 32"):
        lb.mx4_quantize(torch.zeros(4, 0, device="cuda"))
    with pytest.raises(TypeError, match="dtype"):
        lb.mx4_quantize(x.half())
    with pytest.raises(ValueError, match="block axes"):
        lb.mx4_matmul_t(q, lb.mx4_quantize(torch.zeros(4, 32, device="cuda")))
    with pytest.raises(TypeError, match="two microscaled"):
        lb.mx4_matmul_t(x, q)
    with pytest.raises(ValueError, match="bias must hold"):
        lb.mx4_matmul_t(q, q, torch.zeros(5, device="cuda"))
    with pytest.raises(TypeError, match="dtype"):
        lb.mx4_matmul_t(q, q, dtype=torch.float16)
    with pytest.raises(ValueError, match="dy must be"):
        lb.mx4_matmul_dx(x, q)
    with pytest.raises(ValueError, match="last dim"):
        lb.Mx4Linear(q)(torch.zeros(4, 32, device="cuda"))
    with pytest.raises(ValueError, match="contiguous bytes"):
        lb.Mx4Tensor(q.codes, q.scales[:-1], 4, 64)


def test_quant_spelling():
    import loractl_b200 as lb

    assert lb.Quant.parse("MXFP4") is lb.Quant.MXFP4 and lb.quant_value(lb.Quant.MXFP4) == "mxfp4"
    with pytest.raises(ValueError, match="unknown quant"):
        lb.Quant.parse("nvfp4")


def test_refusals_without_a_gpu():
    import loractl_b200 as lb
    from loractl_b200 import _lib as L

    with pytest.raises(RuntimeError, match="CUDA"):
        lb.mx4_quantize(torch.zeros(4, 64))
    lib = L.lib()
    assert lib.lq_mx4_scale_bytes(1, 32) == 1024 and lib.lq_mx4_scale_bytes(129, 288) == 2 * 4 * 512
    assert lib.lq_mx4_scale_bytes(300, 256) == 4 * 2 * 512 and lib.lq_mx4_scale_bytes(0, 32) == 0
    assert lib.lq_mx4_quantize(16, L.LQ_BF16, 1, 48, 48, 16, 16, None) == L.LQ_ERR_INVALID
    assert b"multiple of 32" in lib.lq_last_error()
    assert lib.lq_mx4_quantize(16, 9, 1, 32, 32, 16, 16, None) == L.LQ_ERR_INVALID
    assert lib.lq_mx4_quantize(16, L.LQ_BF16, 2, 32, 16, 16, 16, None) == L.LQ_ERR_INVALID and b"overlap" in lib.lq_last_error()
    assert lib.lq_mx4_quantize(16, L.LQ_BF16, 1, 32, 32, 8, 16, None) == L.LQ_ERR_INVALID and b"aligned" in lib.lq_last_error()
    assert lib.lq_mx4_matmul(16, 16, 1, 16, 16, 1, 32, None, None, L.LQ_F32, None) == L.LQ_ERR_INVALID
    assert lib.lq_mx4_matmul(16, 16, 0, 16, 16, 1, 32, None, None, L.LQ_F32, None) == L.LQ_OK
    assert lib.lq_mx4_dequantize(16, 16, 1, 32, 8, L.LQ_F32, None) == L.LQ_ERR_INVALID
    assert lib.lq_mx4_matmul_dx(16, L.LQ_F32, 1, 16, 16, 4, 32, 16, None, 0, None) == L.LQ_ERR_INVALID
