"""The fused nodes under saved-tensor hooks (non-reentrant checkpoints, offloading, copies of other strides) and under a swap
of `.data`: a backward reads what unpacking gives, at that tensor's address and strides, never the forward's memory, which
may be somebody else's by then.

A hook that gives the same values at the same alignment starts the same kernels on the same numbers, and sums have a fixed
order: gradients are equal bit for bit.  Rows that come back off their 16 bytes take the single-element kernels, whose f32 sums
run in another order: 2^-24 * 64 = 4e-6 of the largest magnitude of either side (twice that between them), and one more rounding
step for gradients held in bf16."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

BF, F = torch.bfloat16, torch.float32
NAMES = ("x", "gate", "y", "shift", "scale", "weight", "post_weight")


def leaves(b, t, h, dtype, mod, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda s, d, std: (torch.randn(*s, generator=g, device="cuda") * std).to(d).requires_grad_(True)
    return {"x": mk((b, t, h), dtype, 1.5), "gate": mk((b, 1, h), mod, 0.4), "y": mk((b, t, h), dtype, 1.0), "shift": mk((b, 1, h), mod, 0.4),
            "scale": mk((b, 1, h), mod, 0.4), "weight": mk((h,), F, 0.3), "post_weight": mk((h,), F, 0.3)}


def seam(v, two=True, norm="zrms", post=True):
    """The operator on copies that die with the call, so that only what the node keeps is left of its inputs."""
    from loractl_b200.block_ops import gated_residual_norm, modulated_zrmsnorm

    c = {k: t * 1 for k, t in v.items()}
    if not two:
        return (modulated_zrmsnorm(c["x"], c["weight"], c["shift"], c["scale"]),)
    return gated_residual_norm(c["x"], c["gate"], c["y"], c["shift"], c["scale"], norm=norm, weight=c["weight"],
                               post_weight=c["post_weight"] if post else None, residual_scale=0.75)


def overwrite(like):
    """Fills memory that has been freed in between (the caching allocator hands it out again by size) with NaN."""
    return [torch.full_like(t, float("nan")) for t in like for _ in range(6)]


def gradients(outs, v):
    seeds = [torch.randn(o.shape, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").to(o.dtype) for o in outs]
    return torch.autograd.grad(outs, list(v.values()), seeds, allow_unused=True)


def padded(t):
    """The same values with rows that start anywhere."""
    wide = t.new_full((*t.shape[:-1], t.shape[-1] + 3), float("nan"))
    wide[..., 1:-2] = t
    return wide[..., 1:-2]


def turned(t):
    """The same values with the last axis strided."""
    return t.movedim(-1, 0).contiguous().movedim(0, -1)


def alike(a, b, exact):
    assert (a is None) == (b is None)
    if a is None:
        return
    assert a.shape == b.shape and a.dtype == b.dtype
    if exact:
        assert torch.equal(a, b)
        return
    step = 2.0 ** -7 if b.dtype == BF else 2.0 ** -22
    a, b, top = a.double(), b.double(), float(b.abs().max())
    assert bool(((a - b).abs() <= 8e-6 * top + step * b.abs()).all())


FORMS = [dict(two=False), dict(), dict(post=False), dict(norm="layer"), dict(norm="layer", post=False)]


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("b,t,h,dtype,mod", [(2, 37, 512, BF, BF), (1, 9, 64, F, F), (3, 20, 521, BF, F), (2, 5, 8200, F, BF)])
def test_seam_under_hooks(form, b, t, h, dtype, mod):
    v = leaves(b, t, h, dtype, mod)
    want = gradients(seam(v, **form), v)
    copies = lambda t: t.clone()
    for pack, unpack, exact in ((copies, copies, True), (copies, padded, False), (copies, turned, True), (lambda t: t.cpu(), lambda t: t.cuda(), True)):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            outs = seam(v, **form)
        junk = overwrite(v.values())
        for ours, ref in zip(gradients(outs, v), want):
            alike(ours, ref, exact or ref is None)
        del junk


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_seam_under_checkpoint_and_offloading(form):
    v = leaves(2, 64, 1024, BF, F)
    want = gradients(seam(v, **form), v)
    outs = checkpoint(lambda *t: seam(dict(zip(NAMES, t)), **form), *v.values(), use_reentrant=False)
    junk = overwrite(v.values())
    for ours, ref in zip(gradients(outs, v), want):
        alike(ours, ref, True)
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        outs = seam(v, **form)
    junk += overwrite(v.values())
    for ours, ref in zip(gradients(outs, v), want):
        alike(ours, ref, True)


@pytest.mark.gpu
def test_seam_after_a_swap_of_data():
    """As torch's own operators: the gradient is that of the values in place when the backward runs (here the same ones)."""
    from loractl_b200.block_ops import gated_residual_norm

    v = leaves(2, 16, 256, BF, F)
    want = gradients(seam(v), v)
    outs = gated_residual_norm(*(v[k] for k in NAMES[:5]), weight=v["weight"], post_weight=v["post_weight"], residual_scale=0.75)
    for t in v.values():
        t.data = t.data.clone()
    junk = overwrite(v.values())
    for ours, ref in zip(gradients(outs, v), want):
        alike(ours, ref, True)
    del junk


@pytest.mark.gpu
def test_seam_refuses_what_a_hook_must_not_give_back():
    v = leaves(2, 8, 64, BF, F)
    for unpack in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t.flatten()[:-1]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
            outs = seam(v)
        with pytest.raises(RuntimeError, match="came back as"):
            gradients(outs, v)

    class Stop(Exception):
        pass

    def stop(t):
        raise Stop

    with pytest.raises(Stop), torch.autograd.graph.saved_tensors_hooks(stop, lambda t: t):
        seam(v)


@pytest.mark.gpu
@pytest.mark.parametrize("n,m,k,r", [(1, 64, 96, 4), (40, 136, 160, 16), (300, 520, 256, 16)])
def test_adapter_under_hooks(n, m, k, r):
    """The microscaled linear with an adapter: every copy has the rows of the original again before the kernels read it."""
    from tests.test_gpu_mx4_lora import site

    _, lora, x, dy = site(n, m, k, r)
    x = x.detach().requires_grad_(True)
    args = [x, lora.delta.lora_a, lora.delta.lora_b]
    want = torch.autograd.grad(lora(x * 1), args, dy)
    copies = lambda t: t.clone()
    for unpack in (copies, padded, turned):
        with torch.autograd.graph.saved_tensors_hooks(copies, unpack):
            y = lora(x * 1)
        junk = overwrite([x])
        for ours, ref in zip(torch.autograd.grad(y, args, dy), want):
            assert torch.equal(ours, ref)
        del junk
    y = checkpoint(lambda t: lora(t * 1), x, use_reentrant=False)
    for ours, ref in zip(torch.autograd.grad(y, args, dy), want):
        assert torch.equal(ours, ref)
    for unpack in (lambda t: t.float(), lambda t: t[..., :-1]):
        with torch.autograd.graph.saved_tensors_hooks(copies, unpack):
            y = lora(x * 1)
        with pytest.raises(RuntimeError, match="came back as"):
            torch.autograd.grad(y, args, dy)


@pytest.mark.gpu
def test_adapter_adds_into_the_flat_buffer_under_a_checkpoint():
    """The unpacked factors are other tensors than the leaves, so autograd accumulates: into the same views, the same sums."""
    import loractl_b200 as lb
    from tests.test_gpu_mx4_lora import site

    _, lora, x, dy = site(40, 136, 160, 16)
    d = lora.delta
    want = torch.autograd.grad(lora(x), [d.lora_a, d.lora_b], dy)
    flat = lb.FlatAdapters(lb.LoraAdapters([d], ["site"]), "cuda")
    flat.zero_grad()
    checkpoint(lora, x, use_reentrant=False).backward(dy)
    for i, p in enumerate((d.lora_a, d.lora_b)):
        assert p.grad.data_ptr() == flat.grad_views(0)[i].data_ptr() and torch.equal(p.grad, want[i])


@pytest.mark.gpu
def test_trunk_block_under_a_checkpoint():
    """A trunk block in bf16 on MXFP4 with adapters and the fused norms, recomputed.  The recomputed forward is the same; the
    gradient of torch's attention may add up in another order, and what it rounds to bf16 then differs by a step of 2^-7 of an element at
    most, which the linear rest of the backward hands on: 2^-6 of the norm."""
    from tests.test_gpu_mx4_training import rel, trunk

    blk, _, adapters, x, tvec, rope = trunk(seed=4)
    params = [p for d in adapters.deltas for p in (d.lora_a, d.lora_b)]
    xs, ts = x.to(BF).requires_grad_(True), tvec.to(BF).requires_grad_(True)
    dy = torch.randn(x.shape, device="cuda").to(BF)
    call = lambda a, c: blk(a, c, rope, None, adapters, "blocks.0")
    plain = call(xs, ts)
    want = torch.autograd.grad(plain, [xs, ts, *params], dy)
    out = checkpoint(call, xs, ts, use_reentrant=False)
    assert torch.equal(out, plain)
    junk = [torch.full((1 << n,), float("nan"), device="cuda") for n in range(4, 20) for _ in range(4)]
    for ours, ref in zip(torch.autograd.grad(out, [xs, ts, *params], dy), want):
        assert bool(torch.isfinite(ours).all()) and rel(ours, ref) <= 2.0 ** -6
    del junk
