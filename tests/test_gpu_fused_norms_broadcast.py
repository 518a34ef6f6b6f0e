"""A trunk block with the fused norms takes the modulation that the block takes without them: one vector for the whole batch too."""
import pytest
import torch
from torch import nn


@pytest.mark.gpu
def test_one_time_vector_for_the_batch():
    """f32 on plain bases, as tests/test_gpu_mx4_training.py compares the two forms: f32 rounding only, 1e-5 of the norm."""
    from tests.test_gpu_mx4_training import rel, trunk

    _, blk, adapters, x, tvec, rope = trunk(seed=5, b=3)
    for _, base in blk.base_linears():
        base.inner.__class__ = nn.Linear
    results = []
    for fused in (False, True):
        blk.fused_norms = fused
        xs, ts = x.clone().requires_grad_(True), tvec[:1].clone().requires_grad_(True)
        out = blk(xs, ts, rope, None, adapters, "blocks.0")
        results.append([out.detach(), *torch.autograd.grad(out, [xs, ts], torch.ones_like(out))])
    for ours, ref in zip(results[1], results[0]):
        assert ours.shape == ref.shape and rel(ours, ref) <= 1e-5
