"""`global_grad_norm`, `clip_grad_norm` and the clipped optimizer step against the formulas in 64 bits: types, ragged and
unaligned tensors, lists longer than one launch, extreme magnitudes, Inf and NaN, in place and to other tensors,
captured calls, the trainer's option, and what is refused.

Tolerances: sums are 64-bit, so the norm is off by its one rounding to f32 (2^-24) plus 2^-53 a term; a clipped value by
the rounding of the factor to f32, of the product, and of the type it is held in (2^-24 + 2^-24, and 2^-8 more in bf16)."""
import pytest
import torch

BF, F = torch.bfloat16, torch.float32


def tensors(sizes, seed=0, spread=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, (n, dt) in enumerate(sizes):
        v = torch.randn(n, generator=g, device="cuda") * (10.0 ** (-(i % 5)) if spread else 1.0)
        out.append(v.to(dt))
    return out


def reference(grads, max_norm=None, scale=1.0):
    total = sum(float(t.double().square().sum()) for t in grads)
    norm = abs(scale) * total ** 0.5
    coef = None if max_norm is None else min(1.0, max_norm / (norm + 1e-6))
    return norm, coef


def near(value, ref, rel):
    return abs(float(value) - ref) <= rel * abs(ref)


LISTS = {
    "one": [(1, F)], "empty_and_one": [(0, F), (1, BF), (0, BF)], "chunk_borders": [(8191, F), (8192, F), (8193, F), (16383, BF), (16385, BF)],
    "factors": [(s, F) for s in (6144 * 16, 16 * 6144, 16 * 1536, 16384 * 16)] * 8, "mixed": [(777, F), (12345, BF), (5, F), (70001, BF), (4, BF)],
    "long": [(1 + 13 * i, F if i % 2 else BF) for i in range(1500)], "large": [(40_000_003, F), (30_000_001, BF)],
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(LISTS))
def test_norm_and_clip_match_the_formula(name):
    import loractl_b200 as lb

    grads = tensors(LISTS[name])
    norm, _ = reference(grads)
    assert near(lb.global_grad_norm(grads), norm, 2.0 ** -23)
    assert near(lb.global_grad_norm(grads, grad_scale=-0.5), norm / 2, 2.0 ** -23)
    for max_norm, scale in ((0.3 * norm, 1.0), (2 * norm + 1, 1.0), (0.1 * norm, 0.25), (0.0, 1.0)):
        n, c = reference(grads, max_norm, scale)
        outs = [torch.full_like(t, 7.0) for t in grads]
        before = [t.clone() for t in grads]
        got = lb.clip_grad_norm(grads, max_norm, out=outs, grad_scale=scale)
        assert near(got, n, 2.0 ** -23) and all(torch.equal(a, b) for a, b in zip(grads, before))
        copies = [t.clone() for t in grads]
        got2 = lb.clip_grad_norm(copies, max_norm, grad_scale=scale)
        assert float(got2) == float(got) and all(torch.equal(a, b) for a, b in zip(copies, outs))
        for t, o in zip(grads, outs):
            ref = t.double() * (scale * c)
            tol = ref.abs() * (2.0 ** -22 + (2.0 ** -8 if t.dtype == BF else 0.0)) + 1e-45
            assert bool(((o.double() - ref).abs() <= tol).all())
            if c == 1.0 and scale == 1.0:
                assert torch.equal(o, t)


@pytest.mark.gpu
def test_unaligned_and_strided_tensors():
    import loractl_b200 as lb

    base = torch.randn(100_000, device="cuda")
    half = torch.randn(100_000, device="cuda").to(BF)
    grads = [base[1:30_000], base[40_003:90_000].view(-1), half[1:50_000], half[60_001:99_999], torch.randn(300, 200, device="cuda").t()]
    norm, coef = reference(grads, 1.0)
    assert near(lb.global_grad_norm(grads), norm, 2.0 ** -23)
    flat = torch.zeros(sum(t.numel() for t in grads if t.dtype == F) + 1, device="cuda")
    flat16 = torch.zeros(sum(t.numel() for t in grads if t.dtype == BF) + 1, dtype=BF, device="cuda")
    outs, at = [], {F: 1, BF: 1}
    for t in grads:
        buf = flat if t.dtype == F else flat16
        outs.append(buf[at[t.dtype]:at[t.dtype] + t.numel()].view(t.shape))
        at[t.dtype] += t.numel()
    lb.clip_grad_norm(grads, 1.0, out=outs)
    for t, o in zip(grads, outs):
        ref = t.double() * coef
        assert bool(((o.double() - ref).abs() <= ref.abs() * (2.0 ** -22 + (2.0 ** -8 if t.dtype == BF else 0.0))).all())
    assert float(flat[0]) == 0 and float(flat16[0]) == 0  # nothing outside the outputs


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,starts", [(BF, 8), (F, 4)])
@pytest.mark.parametrize("size", [1, 6, 33, 8200, 33_000])
def test_every_start_of_source_and_output(dtype, starts, size):
    """Values unscaled (a bound above the norm) and halved (exact): each output is its gradient, its surroundings stay."""
    import loractl_b200 as lb

    room = size + 2 * starts
    src = torch.randn(starts * starts, room, device="cuda").to(dtype)
    dst = torch.full_like(src, 7.0)
    pairs = [(i, i // starts, i % starts) for i in range(starts * starts)]
    grads = [src[i].narrow(0, a, size) for i, a, _ in pairs]
    outs = [dst[i].narrow(0, b, size) for i, _, b in pairs]
    norm = torch.cat(grads).double().norm()
    for factor in (1.0, 0.5):
        got = lb.clip_grad_norm(grads, 1e30, out=outs, grad_scale=factor)
        assert near(got, float(norm) * factor, 2.0 ** -23)
        want = torch.full_like(src, 7.0)
        for i, a, b in pairs:
            want[i].narrow(0, b, size).copy_(grads[i] * factor)
        assert torch.equal(dst, want)
    copy = src.clone()
    lb.clip_grad_norm([copy[i].narrow(0, a, size) for i, a, _ in pairs], 1e30, grad_scale=0.5)
    want = src.clone()
    for i, a, _ in pairs:
        want[i].narrow(0, a, size).mul_(0.5)
    assert torch.equal(copy, want)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-42, 1e-30, 1e30, 3e38])
def test_extreme_magnitudes(size):
    """Squares outside the f32 range; a norm above the largest f32 is Inf and the clip still finite."""
    import loractl_b200 as lb

    g = torch.full((1000,), size, device="cuda")
    norm, coef = reference([g], 1.0)
    got = float(lb.global_grad_norm([g]))
    assert got == float(torch.tensor(norm, dtype=torch.float64).float()) or near(got, norm, 2.0 ** -23)
    lb.clip_grad_norm([g], 1.0)
    ref = size * coef
    assert bool((torch.abs(g.double() - ref) <= 2.0 ** -21 * ref + 1e-44).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("where", [0, 8191, 99_999])
def test_nonfinite_gradients_show(bad, where):
    import loractl_b200 as lb

    g = torch.randn(100_000, device="cuda")
    other = torch.randn(77, device="cuda")
    assert torch.isfinite(lb.global_grad_norm([g, other]))
    g[where] = bad
    assert not torch.isfinite(lb.global_grad_norm([g, other]))
    lb.clip_grad_norm([g, other], 1.0)
    if bad == bad:  # norm Inf: the factor is 0, Inf * 0 is NaN
        assert torch.isnan(g[where]) and int(torch.isnan(g).sum()) == 1 and not other.any()
    else:
        assert torch.isnan(g).all() and torch.isnan(other).all()


@pytest.mark.gpu
def test_determinism_version_counter_streams_and_capture():
    import loractl_b200 as lb

    grads = tensors(LISTS["mixed"] * 50, seed=3)
    first = lb.global_grad_norm(grads)
    assert all(float(lb.global_grad_norm(grads)) == float(first) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert float(lb.global_grad_norm(grads)) == float(first)
    version = grads[0]._version
    outs = [torch.empty_like(t) for t in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = lb.clip_grad_norm(grads, 0.5, out=outs)
    with torch.cuda.graph(graph2 := torch.cuda.CUDAGraph()):
        norm2 = lb.global_grad_norm(grads[::-1])
    for t in grads:
        t.mul_(2.0)
    graph.replay()
    graph2.replay()
    graph.replay()
    ref, coef = reference(grads, 0.5)
    assert near(norm, ref, 2.0 ** -23) and near(norm2, ref, 2.0 ** -23)
    assert near(lb.global_grad_norm(outs), 0.5, 2.0 ** -8)
    lb.clip_grad_norm(grads, 0.5)
    assert grads[0]._version > version + 1 and all(torch.equal(a, b) for a, b in zip(grads, outs))


def adapters():
    import loractl_b200 as lb

    sites = [lb.LoraSite("blocks.0.w1", 64, 96), lb.LoraSite("blocks.0.w2", 96, 64)]
    ad = lb.build_adapters(sites, lb.LoraConfig(rank=4, alpha=8.0, targets=[lb.TargetSpec("blocks")]), "cuda")
    return ad, lb.FlatAdapters(ad, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [0.05, 100.0])
def test_clipped_adamw_matches_torch(max_norm):
    """Three steps against torch's clipping and AdamW on copies; f32 on both sides, 1e-6 of each parameter's change
    budget: an update is at most lr per step whatever the gradient, and its relative error a few 2^-24."""
    import loractl_b200 as lb

    ad, flat = adapters()
    opt = lb.AdamW(flat, weight_decay=0.01)
    copies = [p.detach().clone().requires_grad_(True) for d in ad.deltas for p in (d.lora_a, d.lora_b)]
    ref = torch.optim.AdamW(copies, lr=1e-2, eps=1e-5, weight_decay=0.01)
    g = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(3):
        for p, c in zip([p for d in ad.deltas for p in (d.lora_a, d.lora_b)], copies):
            p.grad.copy_(torch.randn(p.shape, generator=g, device="cuda"))
            c.grad = p.grad * 0.5
        want = torch.nn.utils.clip_grad_norm_(copies, max_norm)
        norm, coef = flat.clip_coefficient(max_norm, 0.5)
        opt.step(1e-2, grad_scale=0.5, skip_flag=flat.flag, clip_coef=coef)
        ref.step()
        assert int(flat.flag) == 0 and abs(float(norm) - float(want)) <= 1e-5 * float(want)
    for p, c in zip([p for d in ad.deltas for p in (d.lora_a, d.lora_b)], copies):
        assert float((p - c).abs().max()) <= 3 * 1e-2 * 1e-4
    # without a factor the step is the unclipped one
    flat.grads.fill_(float("nan"))
    before = flat.params.clone()
    _, coef = flat.clip_coefficient(max_norm)
    opt.step(1e-2, skip_flag=flat.flag, clip_coef=coef)
    assert int(flat.flag) == 1 and torch.equal(flat.params, before)


@pytest.mark.gpu
def test_trainer_clips_the_reduced_gradients():
    from loractl_b200.harness import Trainer
    from tests.test_gpu_harness import batch, make

    runs = {}
    for max_norm in (None, 1e9, 1e-3):
        stack, cfg = make()
        tr = Trainer(stack, lr=1e-3, weight_decay=0.0, max_grad_norm=max_norm)
        tr.step(*batch(cfg))
        runs[max_norm] = (stack.flat.params.clone(), stack.flat.grads.clone(), stack.flat.exp_avg.clone(), tr.grad_norm)
    assert runs[None][3] is None and torch.equal(runs[None][0], runs[1e9][0]) and torch.equal(runs[None][1], runs[1e-3][1])
    grads = runs[None][1].double()
    norm = float(grads.square().sum().sqrt())
    assert near(runs[1e9][3], norm, 2.0 ** -23) and norm > 1e-3
    ref = 0.1 * grads * (1e-3 / (norm + 1e-6))  # the first moment after one step
    assert bool(((runs[1e-3][2].double() - ref).abs() <= 2.0 ** -20 * ref.abs() + 1e-30).all())
    with pytest.raises(ValueError, match="max_grad_norm"):
        Trainer(make()[0], max_grad_norm=-1.0)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    import loractl_b200 as lb

    a, b = torch.ones(10, device="cuda"), torch.ones(10, device="cuda")
    with pytest.raises(TypeError, match="dtype"):
        lb.global_grad_norm([a, b.half()])
    with pytest.raises(RuntimeError, match="one CUDA device"):
        lb.global_grad_norm([a, b.cpu()])
    with pytest.raises(ValueError, match="overlap one another"):
        lb.clip_grad_norm([a, a], 1.0)
    with pytest.raises(ValueError, match="contiguous"):
        lb.clip_grad_norm([torch.ones(4, 4, device="cuda").t()], 1.0)
    with pytest.raises(ValueError, match="same shape"):
        lb.clip_grad_norm([a], 1.0, out=[b[:9]])
    with pytest.raises(ValueError, match="other than its own"):
        lb.clip_grad_norm([a[:5], b[:5]], 1.0, out=[b[:5], a[5:]])
    assert torch.equal(a, torch.ones(10, device="cuda"))
    assert lb.clip_grad_norm([a], 1.0, out=[a]).item() == pytest.approx(10 ** 0.5)
    assert float(lb.global_grad_norm(torch.full((4,), 2.0, device="cuda"))) == 4.0


@pytest.mark.gpu
def test_step_refuses_a_coefficient_that_it_cannot_read():
    import loractl_b200 as lb

    delta = lb.LoraDelta(8, 8, 2, 4.0, device="cuda")
    flat = lb.FlatAdapters(lb.LoraAdapters([delta], ["site"]), "cuda")
    opt, before = lb.AdamW(flat, weight_decay=0.0), flat.params.clone()
    for bad in (torch.ones(()), torch.ones((), device="cuda", dtype=torch.float64), torch.ones(2, device="cuda")):
        with pytest.raises(ValueError, match="clip_coef must be one f32 value"):
            opt.step(1e-3, clip_coef=bad)
    assert opt.steps == 0 and torch.equal(flat.params, before)


def test_refusals_without_a_gpu():
    import loractl_b200 as lb
    from loractl_b200._lib import ext

    _check_outputs = ext().check_outputs
    t = torch.ones(100)
    with pytest.raises(ValueError, match="no gradient"):
        lb.global_grad_norm([])
    with pytest.raises(RuntimeError, match="CUDA device"):
        lb.clip_grad_norm([t], 1.0)
    parts = [t[:10], t[10:30], t[30:30], t[50:]]
    _check_outputs(parts, parts)
    other = torch.ones(100)
    _check_outputs(parts, [other[:10], other[10:30], other[30:30], other[50:]])
    _check_outputs(parts, [t[:10], other[10:30], other[:0], t[50:]])
    _check_outputs([t, t], [other, torch.ones(100)])  # one gradient twice, to two places
    for grads, outs in ((parts, [t[:10], t[9:29], t[30:30], t[50:]]), (parts, [other[:10], t[11:31], t[:0], other[50:]]),
                        ([t, t], [t, other]), ([t[:50], t[50:]], [t[50:], t[:50]]), ([t[:50]], [t[25:75]]), ([t, t[5:10]], [other, t[5:10]])):
        with pytest.raises(ValueError, match="overlap"):
            _check_outputs(grads, outs)


def test_library_refuses_bad_arguments_on_the_host():
    import ctypes as C

    from loractl_b200 import _lib as L

    lib, call = L.lib(), L.lib().lq_grad_norm
    g, n, k = (C.c_void_p * 1)(16), (C.c_int64 * 1)(4), (C.c_int32 * 1)(L.LQ_F32)
    assert call(None, None, None, None, 1, 1.0, 0.0, 16, None, None, None, 0, None) == L.LQ_ERR_INVALID
    assert call(g, None, n, k, 1, 1.0, 0.0, None, None, None, None, 0, None) == L.LQ_ERR_INVALID
    assert b"no output" in lib.lq_last_error()
    assert call(g, g, n, k, 1, 1.0, -1.0, 16, None, None, None, 0, None) == L.LQ_ERR_INVALID
    assert b"max_norm" in lib.lq_last_error()
    k[0] = 9
    assert call(g, None, n, k, 1, 1.0, 0.0, 16, None, None, None, 0, None) == L.LQ_ERR_INVALID
    k[0], n[0] = L.LQ_F32, -1
    assert call(g, None, n, k, 1, 1.0, 0.0, 16, None, None, None, 0, None) == L.LQ_ERR_INVALID
    n[0], g[0] = 4, 2
    assert call(g, None, n, k, 1, 1.0, 0.0, 16, None, None, None, 0, None) == L.LQ_ERR_INVALID
    assert b"aligned" in lib.lq_last_error()
