"""Run-time options reach the microscaled product as they reach the other persistent GEMMs."""
import pytest
import torch

BF = torch.bfloat16


def grids(call):
    """Grid sizes of the kernels that a captured call launches."""
    cu = pytest.importorskip("cuda.bindings.driver")
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()

    def ok(result):
        assert result[0] == cu.CUresult.CUDA_SUCCESS
        return result[1]

    handle = cu.CUgraph(graph.raw_cuda_graph())
    err, _, count = cu.cuGraphGetNodes(handle)
    err, nodes, count = cu.cuGraphGetNodes(handle, count)
    assert err == cu.CUresult.CUDA_SUCCESS
    out = []
    for node in nodes[:count]:
        if ok(cu.cuGraphNodeGetType(node)) == cu.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            out.append(int(ok(cu.cuGraphKernelNodeGetParams(node)).gridDimX))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("adapter", [False, True])
def test_reserved_sms_stay_free(adapter):
    """4096 tokens, 6144 outputs: 384 tiles for 74 pairs.  With 20 SMs reserved the pair kernel's grid is 128 blocks, and the same
    values come out."""
    import loractl_b200 as lb
    from loractl_b200 import _lib as L

    g = torch.Generator(device="cuda").manual_seed(1)
    layer = lb.Mx4Linear(lb.mx4_quantize(torch.randn(6144, 256, generator=g, device="cuda")))
    x = torch.randn(4096, 256, generator=g, device="cuda").to(BF)
    call = layer
    if adapter:
        call = lb.LoraLinear(layer, 4, 8.0, device="cuda")
        with torch.no_grad():
            call.delta.lora_b.normal_()
    with torch.no_grad():
        want = call(x)
        sms = torch.cuda.get_device_properties(0).multi_processor_count
        assert sms // 2 * 2 in grids(lambda: call(x))
        L.check(L.lib().lq_option_set(b"reserve_sms", 20))
        try:
            seen, y = grids(lambda: call(x)), call(x)
        finally:
            L.check(L.lib().lq_option_set(b"reserve_sms", 0))
    assert torch.equal(y, want)
    assert (sms - 20) // 2 * 2 in seen and sms // 2 * 2 not in seen, seen
    lb.check_device_status()
