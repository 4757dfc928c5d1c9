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


@gpu
@pytest.mark.parametrize("heads", [(4, 4), (4, 1)])
def test_gradients_of_queries_alone(heads):
    """frozen keys and values: the launches for their gradients are left out, dq has the bits that it has with them"""
    from lightly_trian_quant_b200 import grad, ops

    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)  # noqa: E731
    q, k, v, do = r(500, heads[0], 64), r(500, heads[1], 64), r(500, heads[1], 64), r(500, heads[0], 64)
    plan = ops.AttnPlan([370, 130], causal=True)
    out, lse = ops.attn_packed(q, k, v, plan, cap=20.0)
    want = ops.attn_packed_bwd(do, q, k, v, out, lse, plan, cap=20.0)
    with torch.enable_grad():
        for need in ((True, False, False), (True, True, False), (False, False, True)):
            leaves = [t.clone().requires_grad_(n) for t, n in zip((q, k, v), need)]
            y = grad.attn_packed(*leaves, plan, cap=20.0)
            before = ops.LAUNCHES
            y.backward(do)
            torch.cuda.synchronize()
            assert ops.LAUNCHES - before == (1 if not any(need[1:]) else 2 if heads[0] == heads[1] else 3)
            for t, n, w in zip(leaves, need, want):
                assert torch.equal(t.grad, w) if n else t.grad is None
    dq, none, nothing = ops.attn_packed_bwd(do, q, k, v, out, lse, plan, cap=20.0, keys=False)
    assert torch.equal(dq, want[0]) and none is None and nothing is None
    given = torch.full_like(q, 7)
    assert ops.attn_packed_bwd(do, q, k, v, out, lse, plan, cap=20.0, grads=(given, None, None), keys=False)[0] is given and torch.equal(given, want[0])
    with pytest.raises(ops.KfError, match="keys"):
        ops.attn_packed_bwd(do, q, k, v, out, lse, plan, cap=20.0, grads=(None, torch.empty_like(k), None), keys=False)
    ops.check_device_error()


@gpu
@pytest.mark.parametrize("R,d", [(300, 96), (9000, 333), (7, 4096), (0, 64)])
def test_gradients_of_rows_alone(R, d):
    """a frozen norm: no column sums, dx has the bits that it has with them"""
    from lightly_trian_quant_b200 import grad, ops

    x, dy, w = torch.randn(R, d, device="cuda"), torch.randn(R, d, device="cuda"), 1 + 0.1 * torch.randn(d, device="cuda")
    y, mean, rstd = ops.layer_norm_fwd(x, w, w, 1e-5)
    want = ops.layer_norm_bwd(dy, x, w, mean, rstd, dres=dy)
    dx, none, nothing = ops.layer_norm_bwd(dy, x, w, mean, rstd, dres=dy, affine=False)
    assert torch.equal(dx, want[0]) and none is None and nothing is None
    with torch.enable_grad():
        for need in ((True, False, False), (True, True, True), (False, False, True)):
            leaves = [t.clone().requires_grad_(n) for t, n in zip((x, w, w), need)]
            out = grad.layer_norm(*leaves, 1e-5)
            before = ops.LAUNCHES
            out.backward(dy)
            torch.cuda.synchronize()
            assert ops.LAUNCHES - before == (0 if R == 0 else 2 if any(need[1:]) else 1)
            assert [t.grad is not None for t in leaves] == list(need)
    ops.check_device_error()


CHOICES = [([1605], 16, 1, False, 3), ([1605] * 8, 16, 1, True, 3), ([130] * 20, 16, 1, False, 2), ([130] * 60, 16, 1, False, 2), ([130] * 60, 16, 1, True, 2), ([130] * 150, 8, 1, False, 2),
           ([1605], 12, 4, True, 3), ([1605] * 4, 12, 4, True, 2), ([130] * 60, 12, 4, True, 2), ([1029, 261, 517, 2053, 133, 1, 1605, 711, 64, 129], 12, 4, True, 3), ([200], 16, 8, False, 2)]


@gpu
@pytest.mark.parametrize("lens,Hq,Hk,causal,kernels", CHOICES, ids=lambda v: f"{len(v)}x{max(v)}" if isinstance(v, list) else str(v))
def test_shared_key_heads_are_split_where_that_is_shorter(lens, Hq, Hk, causal, kernels):
    """the choices of the second launch on 148 SMs, and the workspace that goes with them: 64 KB per key tile and query head of a split, which only batches of few items are"""
    from lightly_trian_quant_b200 import ops

    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the choice depends on the number of SMs")
    q, k = torch.zeros(sum(lens), Hq, 64, dtype=BF, device="cuda"), torch.zeros(sum(lens), Hk, 64, dtype=BF, device="cuda")
    plan = ops.AttnPlan(lens, causal=causal)
    out, lse = ops.attn_packed(q, k, k, plan)
    before = ops.LAUNCHES
    ops.attn_packed_bwd(q, q, k, k, out, lse, plan)
    ops.check_device_error()
    assert ops.LAUNCHES - before == kernels


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16])
def test_split_and_whole_key_heads_against_the_same_reference(dtype):
    """a plan that does not know its lengths splits wherever every query head finds an SM"""
    from lightly_trian_quant_b200 import ops
    from tests.test_attn_pack_gpu import NAMES, case, close, reference, run

    lens, Hq, Hk = [130] * 9, 4, 1
    q, k, v, do = case(lens, lens, Hq, Hk, dtype, 41)
    ref = reference(q, k, v, do, lens, lens, True, None, 0.125, 0.0, None, dtype)
    plan = ops.AttnPlan(lens, causal=True)
    assert plan.k_longest == 130 and plan.k_work == 9 * 132
    for known, kernels in ((True, 2), (False, 3)):
        if not known:
            plan.k_work = plan.k_longest = 0
        before = ops.LAUNCHES
        close(run(q, k, v, do, plan), ref, NAMES)
        assert ops.LAUNCHES - before == 1 + kernels
