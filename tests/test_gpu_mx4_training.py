"""The operators together, as a LoRA training step on a microscaled 4-bit base uses them: the trunk block and the
double-stream stack with MXFP4 linears, fused norms, adapters, the clipped optimizer step, and the step as CUDA graphs.

The twin of the trunk block is plain PyTorch: the same block whose linears multiply `x + (quant(x) - x).detach()` (values
quantised, gradient passed through) with the dequantised weight in f32.  Both sides compute in f32 and differ by ~1e-6
relative; what that can move is an activation next to a rounding border, which then differs by one step of the grid
(at most half of its value).  Eight borders with a relative width of 1e-5 each catch at most ~1e-4 of the elements, so one
product's operand differs by sqrt(1e-4) * 0.5 = 5e-3 relative (Frobenius) at the very worst, five products in a row 2.5e-2,
and a gradient crosses them once more: 5e-2."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantised(x):
    """Plain f32 tensor ops: the values that MXFP4 holds for x."""
    v = x.reshape(-1, 32)
    top = v.abs().amax(-1, keepdim=True)
    unit = torch.exp2((torch.frexp(top)[1] - 3).clamp(-126, 125).float())
    a = v.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.where(top > 0, (torch.round(a / step) * step).clamp(max=6.0) * unit * torch.sign(v), torch.zeros_like(v)).reshape(x.shape)


class TwinLinear(nn.Linear):
    def forward(self, x):
        return nn.functional.linear(x + (quantised(x.detach()) - x.detach()), self.weight, self.bias)


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30))


def trunk(seed=0, features=256, heads=8, kvheads=2, tokens=70, b=2):
    import loractl_b200 as lb
    from loractl_b200 import single_stream as S

    torch.manual_seed(seed)
    cfg = S.MmditConfig(features=features, heads=heads, kvheads=kvheads)
    blk = S.SingleStreamBlock(cfg)
    for p in blk.parameters():
        p.requires_grad_(False)
    for m in (blk.prenorm, blk.postnorm, blk.attn.qnorm, blk.attn.knorm):
        m.scale.normal_(0, 0.1)
    blk.mod_lin.normal_(0, 0.2)
    twin = S.SingleStreamBlock(cfg)
    twin.load_state_dict(blk.state_dict())
    blk, twin = blk.cuda(), twin.cuda()
    assert blk.into_quantized("mxfp4") == (8, 0)
    blk.fused_norms = True
    with torch.no_grad():
        for (_, q), (_, t) in zip(blk.base_linears(), twin.base_linears()):
            lin = TwinLinear(t.d_in, t.d_out, bias=False, device="cuda")
            lin.weight.copy_(q.inner.dequantized_weight())
            t.inner = lin
    adapters = lb.build_adapters(blk.injectable_sites("blocks.0"), lb.LoraConfig(rank=4, alpha=8.0, targets=[lb.TargetSpec(r".*")]),
                                 torch.device("cuda"))
    with torch.no_grad():
        for d in adapters.deltas:
            d.lora_b.normal_(0, 0.05)
    x = torch.randn(b, tokens, features, device="cuda")
    tvec = torch.randn(b, 1, 6 * features, device="cuda") * 0.3
    pos = torch.randint(0, 50, (b, tokens, 3), device="cuda").float()
    return blk, twin, adapters, x, tvec, S.rope_tables(pos, features // heads, cfg.theta)


def test_trunk_block_and_gradients_match_the_twin():
    import loractl_b200 as lb

    blk, twin, adapters, x, tvec, rope = trunk()
    params = [p for d in adapters.deltas for p in (d.lora_a, d.lora_b)]
    dy = torch.randn_like(x)
    got = []
    for model in (blk, twin):
        xs, ts = x.clone().requires_grad_(True), tvec.clone().requires_grad_(True)
        out = model(xs, ts, rope, None, adapters, "blocks.0")
        got.append([out.detach(), *torch.autograd.grad(out, [xs, ts, *params], dy)])
    lb.check_device_status()
    assert rel(got[0][0], got[1][0]) <= 2.5e-2
    for i, (a, b) in enumerate(zip(got[0][1:], got[1][1:])):
        assert torch.isfinite(a).all() and rel(a, b) <= 5e-2, i


def test_fused_norms_are_the_same_function():
    """Plain f32 bases: fused or not, the block differs by f32 rounding only (2^-24 a step; a few hundred steps deep)."""
    blk, twin, adapters, x, tvec, rope = trunk(seed=1)
    outs = []
    for fused in (False, True):
        twin.fused_norms = fused
        for _, t in twin.base_linears():
            t.inner.__class__ = nn.Linear
        xs = x.clone().requires_grad_(True)
        out = twin(xs, tvec, rope, None, adapters, "blocks.0")
        outs.append((out.detach(), torch.autograd.grad(out, xs, torch.ones_like(out))[0]))
    assert rel(outs[1][0], outs[0][0]) <= 1e-5 and rel(outs[1][1], outs[0][1]) <= 1e-5


def test_bf16_step_with_clipping_runs_and_updates():
    """One whole step in bf16: finite gradients for every adapter, a norm that is theirs, parameters that moved, and the
    clipped gradients' norm as the first moment shows it."""
    import loractl_b200 as lb

    blk, _, adapters, x, tvec, rope = trunk(seed=2, features=512, heads=8, kvheads=4, tokens=333)
    flat = lb.FlatAdapters(adapters, "cuda")
    opt = lb.AdamW(flat, weight_decay=0.0)
    flat.zero_grad()
    out = blk(x.bfloat16(), tvec.bfloat16(), rope, None, adapters, "blocks.0")
    out.float().square().mean().backward()
    flat.gather_autograd_grads()
    want = float(flat.grads.double().norm())
    before = flat.params.clone()
    norm, coef = flat.clip_coefficient(want / 4)
    opt.step(1e-3, skip_flag=flat.flag, clip_coef=coef)
    lb.check_device_status()
    ref = want / 4 / (want + 1e-6)  # the 1e-6 of the formula is 2.4e-4 of this norm: 0.24994, not a quarter
    assert abs(float(norm) - want) <= 2 ** -23 * want and abs(float(coef) - ref) <= 2 ** -23 * ref and int(flat.flag) == 0
    assert all(float(p.grad.abs().max()) > 0 for d in adapters.deltas for p in (d.lora_a, d.lora_b))
    assert not torch.equal(before, flat.params) and bool(torch.isfinite(flat.params).all())
    assert abs(float(flat.exp_avg.double().norm()) - 0.1 * want * ref) <= 1e-5 * want


def make_stack(**kw):
    from loractl_b200.harness import BlockConfig, BlockStack

    cfg = BlockConfig(hidden=128, heads=4, mlp=256, img_tokens=64, txt_tokens=16, quant_bits="mxfp4")
    return BlockStack(2, cfg, rank=4, alpha=8.0, device=torch.device("cuda"), seed=5, dtype=torch.bfloat16, **kw), cfg


def test_stack_steps_alike_with_and_without_graphs_and_checkpoints():
    from loractl_b200.harness import Trainer
    from tests.test_gpu_harness import batch

    runs = []
    for kw in ({}, {"graphs": True}, {"grad_checkpointing": False}):
        stack, cfg = make_stack(fused_norms=True)
        tr = Trainer(stack, lr=1e-3, weight_decay=0.0, max_grad_norm=0.01, **kw)
        losses = [tr.step(*batch(cfg, seed=s)) for s in range(3)]
        runs.append((losses, stack.flat.params.clone(), float(tr.grad_norm)))
    for other in runs[1:]:
        assert other[0] == runs[0][0] and torch.equal(other[1], runs[0][1]) and other[2] == runs[0][2]
    assert runs[0][2] > 0


def test_gpt2_on_mxfp4():
    """The text model: quantised projections with biases, loss and adapter gradients, against the twin's linears."""
    import loractl_b200 as lb
    from loractl_b200.gpt2 import Gpt2, Gpt2Config, next_token_loss

    torch.manual_seed(3)
    cfg = Gpt2Config.tiny()
    m, twin = Gpt2(cfg).cuda(), Gpt2(cfg).cuda()
    twin.load_state_dict(m.state_dict())
    assert m.into_quantized("mxfp4") == (8, 0)
    with torch.no_grad():
        for (_, q), (_, t) in zip(m.base_linears(), twin.base_linears()):
            lin = TwinLinear(t.d_in, t.d_out, device="cuda")
            lin.weight.copy_(q.inner.dequantized_weight())
            lin.bias.copy_(t.inner.bias)
            t.inner = lin.requires_grad_(False)
    adapters = lb.build_adapters(m.injectable_sites(), lb.LoraConfig(rank=2, alpha=4.0, targets=[lb.TargetSpec(r".*")]), torch.device("cuda"))
    with torch.no_grad():
        for d in adapters.deltas:
            d.lora_b.normal_(0, 0.05)
    params = [p for d in adapters.deltas for p in (d.lora_a, d.lora_b)]
    ids = torch.randint(0, cfg.vocab_size, (2, 16), device="cuda")
    got = []
    for model in (m, twin):
        logits = model(ids, adapters)
        got.append([logits.detach(), *torch.autograd.grad(next_token_loss(logits, ids), params)])
    assert rel(got[0][0], got[1][0]) <= 5e-2
    for a, b in zip(got[0][1:], got[1][1:]):
        assert rel(a, b) <= 0.1  # two blocks: twice the products of the trunk block


def test_places_that_refuse():
    import loractl_b200 as lb
    from loractl_b200.linear import BaseLinear

    layer = lb.Mx4Linear.from_linear(nn.Linear(64, 48).cuda())
    base = BaseLinear.mx4(layer)
    assert (base.d_in, base.d_out, base.is_quant, base.is_mx4) == (64, 48, False, True)
    with pytest.raises(RuntimeError, match="Mx4"):
        base.as_plain()
    with pytest.raises(RuntimeError, match="Mx4"):
        base.quantize_("mxfp4")
    assert not BaseLinear.plain(nn.Linear(48, 8).cuda()).quantize_("mxfp4")
    with pytest.raises(ValueError, match="take none"):
        make_stack(weight_copies="resident")
    lora = lb.LoraLinear(layer, 4, 8.0, device="cuda")
    x = torch.randn(5, 64, device="cuda")
    assert torch.equal(lora(x), layer(x))  # zero-initialised B
