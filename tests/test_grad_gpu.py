"""The differentiable forms (grad.py): a pre-norm attention block over packed clips against the same block in float64, and their refusals.

Tolerance: the block's intermediate tensors are bf16, u = 2^-8 per rounding.  About ten roundings lie between an input and a result (LayerNorm's output, the
projection, the turn, P, the attention's output, the output projection, and their gradients), independent and of relative size u / sqrt(3) each: 6 u of the
result's root mean square bounds a relative Frobenius error of sqrt(10 / 3) u = 1.8 u with room for the amplification by the softmax (scores of size
2 move by 2 u each: a factor up to 3)."""
import pytest
import torch

from oracle import train_oracle as to

gpu = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _with_grad():
    with torch.enable_grad():                     # modules of the inference path turn it off for the whole process
        yield


def _block(x, w1, b1, wqkv, wout, lens, prefix, pos, table, slopes, cap, low):
    """a pre-norm attention block: low precision through grad, or float64 through the oracle"""
    H = 4
    if low:
        from lightly_trian_quant_b200 import grad, ops

        h = grad.layer_norm(x, w1, b1, 1e-5, BF)
        qkv = (h @ wqkv.to(BF)).view(-1, H + 2 * 2, 64)
        qk = grad.rope_axes(qkv[:, :H + 2], pos, table)
        o = grad.attn_packed(qk[:, :H], qk[:, H:], qkv[:, H + 2:], ops.AttnPlan(lens, causal=True, prefix=prefix), cap=cap, slopes=slopes)
        return x + (o.reshape(-1, H * 64) @ wout.to(BF)).float()
    h = to.layer_norm(x, w1, b1, 1e-5)
    qkv = (h @ wqkv).view(-1, H + 2 * 2, 64)
    angle = torch.cat([pos[:, a:a + 1].double() * torch.tensor(fs, dtype=torch.float64) for a, fs in enumerate(table)], 1)[:, None]
    a, b = qkv[:, :H + 2, :32], qkv[:, :H + 2, 32:]
    qk = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)
    o, _ = to.attn(qk[:, :H], qk[:, H:], qkv[:, H + 2:], lens, lens, causal=True, prefix=prefix, cap=cap, slopes=slopes)
    return x + o.reshape(-1, H * 64) @ wout


@gpu
def test_a_block_and_its_gradients():
    from lightly_trian_quant_b200 import ops

    g = torch.Generator().manual_seed(5)
    lens, prefix, d = [137, 40, 261], [5, 5, 5], 192
    freqs = [[100.0 ** -(i / 11) for i in range(11)], [100.0 ** -(i / 11) for i in range(11)], [1.0 / (i + 1) for i in range(10)]]
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    data = dict(x=r(sum(lens), d), w1=1 + 0.1 * r(d), b1=0.1 * r(d), wqkv=(r(d, 8 * 64) / d ** 0.5).to(BF).float(), wout=(r(4 * 64, d) / 16).to(BF).float())
    pos = torch.randint(0, 40, (sum(lens), 3), generator=g)
    slopes, dy = torch.tensor([0.01, 0.0, 0.05, 0.1]), r(sum(lens), d)
    leaves = {n: t.cuda().requires_grad_() for n, t in data.items()}
    y = _block(*leaves.values(), lens, prefix, pos.cuda(), ops.RopeTable(freqs, 64), slopes.cuda(), 20.0, True)
    y.backward(dy.cuda())
    ops.check_device_error()
    ref = {n: t.double().requires_grad_() for n, t in data.items()}
    want = _block(*ref.values(), lens, prefix, pos, freqs, slopes, 20.0, False)
    want.backward(dy.double())
    rel = lambda a, b: ((a.double().cpu() - b).norm() / b.norm()).item()  # noqa: E731
    errors = {"y": rel(y.detach() - leaves["x"].detach(), (want - ref["x"]).detach()), **{n: rel(t.grad, ref[n].grad) for n, t in leaves.items()}}
    assert max(errors.values()) < 6 * 2 ** -8, errors
    assert all(t.grad.dtype == t.dtype for t in leaves.values())


@gpu
def test_gradients_that_are_expanded_or_permuted():
    from lightly_trian_quant_b200 import grad, ops

    x = torch.randn(40, 96, device="cuda", requires_grad=True)
    w = torch.ones(96, device="cuda", requires_grad=True)
    grad.layer_norm(x, w, None, 1e-5).sum().backward()                         # an expanded gradient
    # dy = 1: g = w = 1, dx = rstd (1 - 1 - xh mean(xh)), mean(xh) = 0 up to rounding
    assert x.grad.abs().max() < 1e-4 and torch.isfinite(w.grad).all()
    q = torch.randn(40, 2, 64, device="cuda").bfloat16().requires_grad_()
    out = grad.attn_packed(q, q, q, ops.AttnPlan([40]))
    out.permute(2, 0, 1).float().square().sum().backward()
    assert torch.isfinite(q.grad).all() and q.grad.abs().max() > 0
    z = torch.randn(40, 2, 64, device="cuda", requires_grad=True)
    pos = torch.arange(40, device="cuda")[:, None]
    y = grad.rope_axes(z, pos, ops.RopeTable([[0.1] * 32], 64))
    y.transpose(0, 1).reshape(-1).dot(y.detach().transpose(0, 1).reshape(-1)).backward()      # the gradient of |y|^2 / 2 turned back is z
    assert torch.allclose(z.grad, z, atol=1e-5)


@gpu
def test_no_autograd_inside_a_capture():
    from lightly_trian_quant_b200 import grad, ops

    x, w = torch.randn(8, 64, device="cuda", requires_grad=True), torch.ones(64, device="cuda")
    q = torch.randn(8, 1, 64, device="cuda").bfloat16().requires_grad_()
    plan, pos, table = ops.AttnPlan([8]), torch.zeros(8, 1, dtype=torch.int32, device="cuda"), ops.RopeTable([[1.0]], 64)
    calls = (lambda: grad.layer_norm(x, w, w, 1e-5), lambda: grad.attn_packed(q, q, q, plan), lambda: grad.rope_axes(q, pos, table))
    eager = [f() for f in calls]
    kept = {}
    with torch.no_grad():
        calls[0]()                                                             # no gradient wanted: like the operator
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for f in calls:
            with pytest.raises(ops.KfError, match="capture"):
                f()
        with torch.no_grad():
            kept["y"] = calls[0]()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept["y"], eager[0].detach())
    eager[0].sum().backward()
    ops.check_device_error()


@gpu
def test_slopes_have_no_gradient():
    from lightly_trian_quant_b200 import grad, ops

    q = torch.randn(8, 1, 64, device="cuda").bfloat16()
    with pytest.raises(ops.KfError, match="slopes"):
        grad.attn_packed(q, q, q, ops.AttnPlan([8]), slopes=torch.zeros(1, device="cuda", requires_grad=True))


def test_cpu_tensors_are_refused():
    from lightly_trian_quant_b200 import grad, ops

    x = torch.randn(8, 64, requires_grad=True)
    with pytest.raises(ops.KfError):
        grad.layer_norm(x, torch.ones(64), None, 1e-5)
    q = torch.randn(8, 1, 64).bfloat16()
    with pytest.raises(ops.KfError):
        grad.attn_packed(q, q, q, ops.AttnPlan([8], device="cpu"))
