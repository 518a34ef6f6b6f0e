"""Clipping at the edges of its factor's range and of its list of tensors, beside tests/test_gpu_grad_norm.py."""
import pytest
import torch

BF, F = torch.bfloat16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("exponent", [-126, -127, -130, -140])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -13, 2.0 ** -10])
def test_factors_next_to_a_power_of_two(dtype, exponent, small):
    """Factors of 2^exponent and a little below: below 2^-126 they are held as m * 2^e, and the m of the second (1 - 2^-27)
    rounds to one.  In place that must not read as "nothing to scale".  The factor is off by its rounding to f32 (2^-24), the product by
    another, and by the type's own (2^-9 in bf16, for which 2^-8 stands)."""
    import loractl_b200 as lb

    top = 2.0 ** 100
    g = torch.tensor([top, -top * small, 0.0, top * small / 8], device="cuda", dtype=dtype)
    norm = float(g.double().square().sum()) ** 0.5
    max_norm = 2.0 ** (100 + exponent)
    want = g.double() * min(1.0, max_norm / (norm + 1e-6))
    out = torch.empty_like(g)
    lb.clip_grad_norm([g], max_norm, out=[out])
    lb.clip_grad_norm([g], max_norm)
    rel = 2.0 ** -23 + (2.0 ** -8 if dtype == BF else 2.0 ** -24)
    for got in (out, g):
        assert bool(((got.double() - want).abs() <= rel * want.abs()).all()), (got, want)
