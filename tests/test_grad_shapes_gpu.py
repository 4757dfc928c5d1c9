"""Gradients as autograd hands them on: views into others, at any offset."""
import pytest
import torch

gpu = pytest.mark.gpu
BF = torch.bfloat16


@gpu
@pytest.mark.parametrize("odd", [1, 3, 8])
def test_gradients_that_start_anywhere(odd):
    """an output that was flattened and put behind something else gets a view of the whole gradient, contiguous, at an address that is a multiple of two bytes only: the same
    gradients as from a tensor of its own"""
    from lightly_trian_quant_b200 import grad, ops

    g = torch.Generator(device="cuda").manual_seed(odd)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)  # noqa: E731
    T, H = 70, 2
    q, w, b = r(T, H, 64), torch.ones(H * 64, device="cuda"), torch.zeros(H * 64, device="cuda")
    pos, plan = torch.arange(T, device="cuda")[:, None], ops.AttnPlan([50, 20], causal=True)
    half, pairs = ops.RopeTable([[0.1] * 32], 64), ops.RopeTable([[0.1] * 20], 64, interleaved=True)
    calls = (lambda x: grad.attn_packed(x, x, x, plan), lambda x: grad.rope_axes(x, pos, half), lambda x: grad.rope_axes(x, pos, pairs),
             lambda x: grad.layer_norm(x.view(T, H * 64), w, b, 1e-5))
    dy, front = r(T * H * 64), r(odd)
    with torch.enable_grad():
        for call in calls:
            x, z = q.clone().requires_grad_(), q.clone().requires_grad_()
            call(x).flatten().backward(dy)
            torch.cat((front.requires_grad_(), call(z).flatten())).backward(torch.cat((front.detach(), dy)))
            assert torch.equal(x.grad, z.grad) and x.grad.any()
            front = front.detach()
    ops.check_device_error()
