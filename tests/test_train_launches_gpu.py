"""What the operators for training launch: ops.LAUNCHES against the kernels of a captured graph."""
import pytest
import torch

gpu = pytest.mark.gpu
BF = torch.bfloat16


def _kernels(call):
    """call() captured -> (kernels in the graph, what ops.LAUNCHES counted)"""
    from cuda.bindings import runtime as rt

    from lightly_trian_quant_b200 import ops

    call()                                                        # attributes of the kernels are set by their first launch
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    before = ops.LAUNCHES
    with torch.cuda.graph(graph):
        kept = call()
    counted = ops.LAUNCHES - before
    raw = rt.cudaGraph_t(init_value=graph.raw_cuda_graph())
    err, _, n = rt.cudaGraphGetNodes(raw)
    assert int(err) == 0
    err, nodes, _ = rt.cudaGraphGetNodes(raw, n)
    assert int(err) == 0
    kernels = sum(rt.cudaGraphNodeGetType(node)[1] == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for node in nodes)
    graph.reset()
    del kept
    ops.check_device_error()
    return kernels, counted


@gpu
@pytest.mark.parametrize("lens,heads,kernels", [([200], (4, 4), 2), ([200], (4, 1), 3), ([130] * 400, (4, 2), 2), ([0], (4, 2), 0)], ids=str)
def test_launches_of_the_packed_attention(lens, heads, kernels):
    """two kernels for the gradients, three where query heads that share a key head are items of their own"""
    from lightly_trian_quant_b200 import ops

    q = torch.randn(sum(lens), heads[0], 64, device="cuda").to(BF)
    k = torch.randn(sum(lens), heads[1], 64, device="cuda").to(BF)
    plan = ops.AttnPlan(lens)
    out, lse = ops.attn_packed(q, k, k, plan)
    assert _kernels(lambda: ops.attn_packed_bwd(q, q, k, k, out, lse, plan)) == (kernels, kernels)
    if kernels:
        assert _kernels(lambda: ops.attn_packed(q, k, k, plan)) == (1, 1)


@gpu
def test_launches_of_the_row_operators():
    from lightly_trian_quant_b200 import ops

    x, w = torch.randn(40, 96, device="cuda"), torch.ones(96, device="cuda")
    y, mean, rstd = ops.layer_norm_fwd(x, w, w, 1e-5)
    assert _kernels(lambda: ops.layer_norm_fwd(x, w, w, 1e-5)) == (1, 1)
    assert _kernels(lambda: ops.layer_norm_bwd(y, x, w, mean, rstd)) == (2, 2)
    assert _kernels(lambda: ops.layer_norm_bwd(y[:0], x[:0], w, mean[:0], rstd[:0])) == (0, 0)       # two memory sets
    table, pos = ops.RopeTable([[1.0]], 96), torch.zeros(40, 1, dtype=torch.int32, device="cuda")
    assert _kernels(lambda: ops.rope_axes(x.view(40, 1, 96), pos, table)) == (1, 1)
