"""The adapter's node in captures: beside a living eager graph of the same leaves, and on a stream that is not the eager one."""
import subprocess
import sys

import pytest

BESIDE_EAGER = """
import torch
import loractl_b200 as lb
torch.manual_seed(0)
x = torch.randn(40, 64, device="cuda").bfloat16().requires_grad_(True)
def site():
    lora = lb.LoraLinear(lb.Mx4Linear(lb.mx4_quantize(torch.randn(32, 64, device="cuda"))), 4, 8.0, device="cuda")
    with torch.no_grad():
        lora.delta.lora_b.normal_()
    return lora
plain, flat = site(), site()
dy = torch.randn(40, 32, device="cuda").bfloat16()  # torch's generator stays in the capture that an error ends
buffers = lb.FlatAdapters(lb.LoraAdapters([flat.delta], ["site"]), "cuda")
for lora in (plain, flat):
    leaves = [x, lora.delta.lora_a, lora.delta.lora_b]
    want = torch.autograd.grad(plain(x), [x, plain.delta.lora_a, plain.delta.lora_b], dy) if lora is plain else None
    living = lora(x)
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            lora(x).sum().backward()
    except RuntimeError as e:
        assert "capture" in str(e), e
    torch.cuda.synchronize()
    if want is not None:
        x.grad = lora.delta.lora_a.grad = lora.delta.lora_b.grad = None
        for a, b in zip(torch.autograd.grad(living, leaves, dy), want):
            assert torch.equal(a, b)
    else:
        buffers.zero_grad()
        living.backward(dy)
        assert bool(torch.isfinite(buffers.grads).all()) and float(buffers.grads.abs().max()) > 0
    assert bool(torch.isfinite(lora(x)).all())
lb.check_device_status()
print("usable")
"""


@pytest.mark.gpu
def test_capture_beside_a_living_eager_graph():
    """Torch's error about the capture or a capture that holds; the process, the context and the eager graph stay usable."""
    from tests.conftest import ROOT

    r = subprocess.run([sys.executable, "-c", BESIDE_EAGER], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "usable" in r.stdout, r.stdout[-1000:] + r.stderr[-2000:]
