"""y of a microscaled site with an adapter is rounded once, whichever kernels its number of tokens takes: product, bias and delta are
added up in f32.  The numbers are whole or halves, exact in every format on the way, so the values are compared for equality; a
product rounded to bf16 before the delta comes (257 -> 256, 257.5 -> 258) gives others."""
import pytest
import torch

BF = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("n,m", [(1, 8), (1, 6152), (16, 136), (40, 520), (77, 6144), (128, 264), (200, 1000), (1000, 72), (2000, 2048)])
@pytest.mark.parametrize("bias,want", [(None, 258.0), (0.5, 258.0), (2.0, 260.0), (-514.0, -256.0)])
def test_one_rounding(n, m, bias, want):
    import loractl_b200 as lb

    k = 96
    w = torch.zeros(m, k, device="cuda")
    w[:, :64] = 4.0
    w[:, 70] = 1.0  # sums to 257
    b = None if bias is None else torch.full((m,), bias, device="cuda")
    lora = lb.LoraLinear(lb.Mx4Linear(lb.mx4_quantize(w), b), 4, 4.0, device="cuda")
    with torch.no_grad():
        lora.delta.lora_a.zero_()[0, 0] = 1.0
        lora.delta.lora_b.zero_()[0] = 1.0  # a delta of one
    x = torch.ones(n, k, device="cuda", dtype=BF)
    y = lora(x)
    exact = 257.0 + (bias or 0.0) + 1.0
    assert float(torch.tensor(exact).to(BF)) == want
    assert y.grad_fn.name() == "Mx4LoraBackward" and bool((y == want).all())
    lb.check_device_status()
