"""The operators for training on tensors of more than 2^31 elements: what lies behind has the bits that it has alone."""
import pytest
import torch

gpu = pytest.mark.gpu
BF = torch.bfloat16


def _filled(*shape):
    """normal numbers, in pieces: a generator's intermediate would be twice as large"""
    t = torch.empty(*shape, dtype=BF, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for part in t.split(1 << 16):
        part.normal_(generator=g)
    return t


@pytest.fixture(autouse=True)
def _room():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("shared", [1, 4])
def test_packed_attention(shared):
    from lightly_trian_quant_b200 import ops

    H, lens = 64, [131] * 4000 + [77, 300]
    T = sum(lens)
    x = _filled(T, H, 64)
    assert x.numel() > 2 ** 31
    k = x[:, :H // shared]
    plan = ops.AttnPlan(lens, causal=True)
    out, lse = ops.attn_packed(x, k, k, plan)
    grads = ops.attn_packed_bwd(x, x, k, k, out, lse, plan)
    ops.check_device_error()
    for first, part in ((T - 377, [77, 300]), (131 * 3977, [131] * 2)):
        rows = slice(first, first + sum(part))
        q1, k1, alone = x[rows].clone(), k[rows].clone(), ops.AttnPlan(part, causal=True)
        alone.k_work, alone.k_longest = plan.k_work, plan.k_longest            # the same choice of whole key heads
        o1, l1 = ops.attn_packed(q1, k1, k1, alone)
        assert torch.equal(out[rows], o1) and torch.equal(lse[:, rows], l1)
        for a, b in zip(grads, ops.attn_packed_bwd(q1, q1, k1, k1, o1, l1, alone)):
            assert torch.equal(a[rows], b)
    ops.check_device_error()


@gpu
def test_rotary_positions_and_layer_norm():
    from lightly_trian_quant_b200 import ops

    T, H, D = 270_000, 64, 128
    x = _filled(T, H, D)
    assert x.numel() > 2 ** 31
    pos, table = torch.arange(T, device="cuda")[:, None], ops.RopeTable([[1.0 / (i + 1) for i in range(64)]], D)
    y = ops.rope_axes(x, pos, table)
    rows = slice(T - 5000, T)
    assert torch.equal(y[rows], ops.rope_axes(x[rows].clone(), pos[rows].clone(), table))
    del y
    for d in (1024, 999):                                          # aligned rows and others
        R = x.numel() // d
        xs, w = x.view(-1)[:R * d].view(R, d), 1 + 0.1 * torch.randn(d, device="cuda")
        y, mean, rstd = ops.layer_norm_fwd(xs, w, w, 1e-5)
        dx, dw, _ = ops.layer_norm_bwd(y, xs, w, mean, rstd)
        tail = slice(R - 4000, R)
        x1 = xs[tail].clone()
        y1, m1, r1 = ops.layer_norm_fwd(x1, w, w, 1e-5)
        assert torch.equal(y[tail], y1) and torch.equal(mean[tail], m1) and torch.equal(rstd[tail], r1)
        assert torch.equal(dx[tail], ops.layer_norm_bwd(y1, x1, w, m1, r1)[0]) and torch.isfinite(dw).all()
        del y, dx
    ops.check_device_error()
