"""`clip_grad_norm` takes gradients: parameters, which torch's function of that name takes, would be scaled themselves."""
import pytest
import torch

import loractl_b200 as lb


def test_parameters_are_refused():
    lin = torch.nn.Linear(8, 4)
    grads = [torch.ones_like(p) for p in lin.parameters()]
    for call in (lambda: lb.clip_grad_norm(lin.parameters(), 1.0), lambda: lb.clip_grad_norm(grads, 1.0, out=list(lin.parameters()))):
        with pytest.raises(RuntimeError, match="not parameters"):
            call()
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA device"):  # as torch: allowed there
        lb.clip_grad_norm(lin.parameters(), 1.0)


@pytest.mark.gpu
def test_gradients_with_a_graph_and_parameters_without_grad_mode():
    lin = torch.nn.Linear(64, 4).cuda()
    before = [p.detach().clone() for p in lin.parameters()]
    with pytest.raises(RuntimeError, match="not parameters"):
        lb.clip_grad_norm(lin.parameters(), 1e-3)
    assert all(torch.equal(p, b) for p, b in zip(lin.parameters(), before))
    x = torch.randn(5, 64, device="cuda")
    grads = torch.autograd.grad(lin(x).square().sum(), list(lin.parameters()), create_graph=True)
    norm = float(sum(g.double().square().sum() for g in grads)) ** 0.5
    assert abs(float(lb.clip_grad_norm(list(grads), norm / 2)) - norm) <= 2.0 ** -23 * norm  # no leaves: gradients of create_graph
    with torch.no_grad():
        lb.clip_grad_norm(list(lin.parameters()), 1e-3)
    assert float(sum(p.double().square().sum() for p in lin.parameters())) ** 0.5 <= 1.001e-3
