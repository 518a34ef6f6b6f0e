"""Which outputs `clip_grad_norm` takes beside strided gradients: what counts is the memory that a gradient spans."""
import pytest
import torch

from loractl_b200._lib import ext


def test_a_broadcast_gradient_spans_one_row():
    """Nothing behind the one row (or value) that it repeats is the gradient's."""
    t = torch.zeros(4096)
    check = ext().check_outputs
    check([t[:1].expand(1000)], [t[1:1001]])
    check([t[:8].expand(100, 8)], [t[8:808].view(100, 8)])
    check([t[:8].expand(100, 8), t[808:1000]], [t[8:808].view(100, 8), t[1000:1192]])
    with pytest.raises(ValueError, match="overlap"):
        check([t[:8].expand(100, 8)], [t[4:804].view(100, 8)])


def test_a_strided_gradient_spans_its_last_element():
    """numel elements from its start would end before it does."""
    t = torch.zeros(4096)
    check = ext().check_outputs
    every4 = t[:400:4]  # elements 0 .. 396
    check([every4], [t[397:497]])
    for at in (396, 300, 150):
        with pytest.raises(ValueError, match="overlap"):
            check([every4], [t[at:at + 100]])
    columns = t[:1000].view(10, 100)[:, 20:30]  # 20 .. 929
    check([columns], [t[930:1030].view(10, 10)])
    with pytest.raises(ValueError, match="overlap"):
        check([columns], [t[929:1029].view(10, 10)])
    check([columns], [t[20:120].view(10, 10)])  # its own memory, from the same start
    check([t[:0:4], columns], [t[:0], torch.zeros(10, 10)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_broadcast_gradients_are_clipped_to_what_lies_behind_them(dtype):
    """f32 rounds the factor and the product (2^-23 together), bf16 the value once more (2^-8)."""
    import loractl_b200 as lb

    g = torch.Generator(device="cuda").manual_seed(3)
    t = torch.randn(4096, generator=g, device="cuda").to(dtype)
    one, row, cols = t[:1].expand(1000), t[1:9].expand(40, 8), t[16:1016].view(10, 100)[:, 3:9]
    outs = [torch.empty(1000, device="cuda", dtype=dtype), t[1100:1420].view(40, 8), t[2000:2060].view(10, 6)]
    grads = [one, row, cols]
    ref = [v.double() for v in grads]
    norm = sum(float(v.square().sum()) for v in ref) ** 0.5
    got = lb.clip_grad_norm(grads, norm / 3, out=outs)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    for o, r in zip(outs, ref):
        want = r * (norm / 3 / (norm + 1e-6))
        assert bool(((o.double() - want).abs() <= (2.0 ** -22 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) * want.abs()).all())
