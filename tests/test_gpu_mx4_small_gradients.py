"""The f32 gradient through a microscaled weight down to the smallest numbers: an element of dy goes in as three bf16 terms, and bf16
ends at 2^-133, so what an element has below that is cut; all else is exact.  With a unit weight the output is the sum of an
element's terms: equal to it down to 2^-109 (24 bits above 2^-133), and off by less than 2^-133 below."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 400])
@pytest.mark.parametrize("exponent", [0, -60, -109, -110, -118, -126, -132, -140])
def test_terms_of_small_elements(n, exponent):
    import loractl_b200 as lb

    w = lb.mx4_quantize(torch.eye(128, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(2)
    v = (torch.rand(n, 128, generator=g, device="cuda", dtype=torch.float64) + 1) * 2.0 ** exponent
    dy = (v * torch.where(torch.rand(n, 128, generator=g, device="cuda") < 0.5, -1.0, 1.0)).float()
    dx = lb.mx4_matmul_dx(dy, w)
    if exponent >= -109:
        assert torch.equal(dx, dy)
    assert bool(((dx.double() - dy.double()).abs() < 2.0 ** -133).all())
    assert torch.equal(lb.mx4_matmul_dx(dy.bfloat16(), w), dy.bfloat16())
