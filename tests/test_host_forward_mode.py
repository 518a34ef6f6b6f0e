"""The fused nodes have reverse-mode derivatives only: a tensor that carries a forward-mode tangent is refused (its derivative
would be dropped in silence), before anything looks at a device."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from loractl_b200 import _lib as L

NAMES = ("x", "gate", "y", "shift", "scale", "weight", "post_weight")


def shapes(h=32):
    return {k: torch.ones(2, 4, h) if k in "xy" else torch.ones(h) if "weight" in k else torch.ones(2, 1, h) for k in NAMES}


@pytest.mark.parametrize("name", NAMES)
def test_residual_norm(name):
    with fwad.dual_level():
        v = shapes()
        v[name] = fwad.make_dual(v[name], torch.ones_like(v[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            L.ext().residual_norm(*(v[k] for k in NAMES), False, 1.0, 1e-5)


@pytest.mark.parametrize("no_grad", [False, True])
def test_prenorm(no_grad):
    from loractl_b200.block_ops import modulated_zrmsnorm

    v = shapes()
    with fwad.dual_level(), torch.set_grad_enabled(not no_grad):
        x = fwad.make_dual(v["x"], torch.ones_like(v["x"]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            modulated_zrmsnorm(x, None, v["shift"], v["scale"])
    with pytest.raises(RuntimeError, match="CUDA device"):  # without a tangent: the next check
        modulated_zrmsnorm(v["x"], None, v["shift"], v["scale"])


def test_microscaled_linear():
    codes, scales, x = torch.zeros(8, 16, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8), torch.ones(3, 32)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            L.ext().mx4_linear(dual(x), codes, scales, 8, 32, None)
        for name in "xab":
            v = {"x": x, "a": torch.ones(32, 4), "b": torch.ones(4, 8)}
            v[name] = dual(v[name])
            with pytest.raises(NotImplementedError, match="forward-mode"):
                L.ext().mx4_lora_linear(v["x"], codes, scales, 8, 32, None, v["a"], v["b"], 1.0, codes, None, None)


@pytest.mark.gpu
def test_backward_passes():
    """A tangent on an output's gradient (forward over reverse) is refused too; without one the same calls run."""
    import loractl_b200 as lb
    from loractl_b200.block_ops import modulated_zrmsnorm

    x = torch.randn(2, 4, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    v = torch.zeros(2, 1, 32, device="cuda")
    layer = lb.Mx4Linear(lb.mx4_quantize(torch.randn(8, 32, device="cuda")))
    lora = lb.LoraLinear(layer, 4, 8.0, device="cuda")
    for call in (lambda: modulated_zrmsnorm(x, None, v, v), lambda: layer(x), lambda: lora(x)):
        y = call()
        torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
        with fwad.dual_level():
            dy = fwad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, x, dy)
