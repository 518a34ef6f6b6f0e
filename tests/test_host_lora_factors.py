"""Factors that the operand mirror's kernels would misread (other types, strides, shapes) are refused on the host: a bf16 factor
holds half of the bytes that they read."""
import pytest
import torch

from loractl_b200 import quant as Q


def test_mirror_refuses_what_it_would_misread():
    a, b = torch.zeros(64, 4), torch.zeros(4, 32)
    calls = (lambda a, b: Q.lora_mirror(a, b), lambda a, b: Q.lora_mirror_batch([(a, b, torch.zeros(8, dtype=torch.uint8))]))
    for call in calls:
        for bad in ((a.bfloat16(), b), (a, b.bfloat16()), (a.double(), b.double())):
            with pytest.raises(TypeError, match="must be f32"):
                call(*bad)
        for bad in ((torch.zeros(4, 64).t(), b), (a, torch.zeros(32, 4).t()), (a, b[:3]), (a[:, 0], b)):
            with pytest.raises(ValueError, match="contiguous"):
                call(*bad)
        with pytest.raises(RuntimeError, match="CUDA"):
            call(a, b)


@pytest.mark.gpu
def test_adapters_cast_to_bf16_are_refused():
    import loractl_b200 as lb
    from loractl_b200 import _lib as L

    x = torch.randn(5, 64, device="cuda").bfloat16()
    lin = torch.nn.Linear(64, 32).cuda()
    for base in (lb.Mx4Linear.from_linear(lin), lb.QuantLinear.from_linear(lin, 4)):
        lora = lb.LoraLinear(base, 4, 8.0, device="cuda")
        y, mirror = lora(x), lora.delta.operand_mirror()
        lora.delta.to(torch.bfloat16)
        with pytest.raises(TypeError, match="must be f32"):
            lora(x)
    w = lora.delta.lora_a, lora.delta.lora_b
    q = lb.Mx4Linear.from_linear(lin).weight
    with pytest.raises(TypeError, match="must be f32"):
        L.ext().mx4_lora_linear(x, q.codes, q.scales, 32, 64, None, *w, 1.0, mirror, None, None)
    assert y.shape == (5, 32)
