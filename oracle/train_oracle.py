"""CPU oracle of the operators for training: test infrastructure, not product code.  Float64 torch, from the definitions; gradients by differentiation."""
from __future__ import annotations

import torch


def layer_norm(x, w, b, eps):
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    return (x - mean) / (var + eps).sqrt() * w + (0.0 if b is None else b)


def layer_norm_grads(x, w, b, eps, dy):
    """-> y, dx, dw, db in float64"""
    x, w = x.double().requires_grad_(), w.double().requires_grad_()
    b = torch.zeros_like(w).requires_grad_() if b is None else b.double().requires_grad_()
    with torch.enable_grad():
        y = layer_norm(x, w, b, eps)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy.double()))


def rope(x, pos, freqs, interleaved=False, inverse=False):
    """x [..., T, H, D], pos [T, axes], freqs per axis -> the turned x in float64"""
    x, pos = x.double(), pos.double()
    angle = torch.cat([pos[:, a:a + 1] * torch.tensor(fs, dtype=torch.float64) for a, fs in enumerate(freqs)], 1)[:, None]
    P = angle.shape[-1]
    sin, cos = torch.sin(angle) * (-1 if inverse else 1), torch.cos(angle)
    y = x.clone()
    a, b = (x[..., 0:2 * P:2], x[..., 1:2 * P:2]) if interleaved else (x[..., :P], x[..., P:2 * P])
    at = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    y[..., at[0]], y[..., at[1]] = a * cos - b * sin, b * cos + a * sin
    return y


def attn_sees(lq, lk, causal, prefix):
    """[lq, lk] truth values: query i, at position i + lk - lq, sees key j"""
    i, j = torch.arange(lq)[:, None] + (lk - lq), torch.arange(lk)[None]
    return ((j <= i) | (j < prefix)) if causal else torch.ones(lq, lk, dtype=torch.bool)


def attn(q, k, v, q_lens, k_lens, *, causal=False, prefix=None, scale=0.125, cap=0.0, slopes=None):
    """q [Tq, Hq, D], k, v [Tk, Hk, D] in float64 -> out [Tq, Hq, D], lse [Hq, Tq]; rows that see nothing: 0 and -inf.  Differentiable."""
    share = q.shape[1] // k.shape[1]
    outs, lses = [], []
    q0 = k0 = 0
    for d, (lq, lk) in enumerate(zip(q_lens, k_lens)):
        qd, kd, vd = q[q0:q0 + lq], k[k0:k0 + lk].repeat_interleave(share, 1), v[k0:k0 + lk].repeat_interleave(share, 1)
        s = torch.einsum("ihd,jhd->hij", qd, kd) * scale
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            far = (torch.arange(lq)[:, None] + (lk - lq) - torch.arange(lk)[None]).abs()
            s = s - slopes.double()[:, None, None] * far
        sees = attn_sees(lq, lk, causal, prefix[d] if prefix else 0)
        any_ = sees.any(1)
        s = torch.where(sees, s, torch.full_like(s, -1e300))
        p = torch.softmax(s, -1) * sees if lk else s
        outs.append(torch.einsum("hij,jhd->ihd", p, vd) * any_[:, None, None])
        z = torch.logsumexp(s, -1) if lk else s.new_zeros(s.shape[:2])
        lses.append(torch.where(any_, z, torch.full_like(z, float("-inf"))))
        q0, k0 = q0 + lq, k0 + lk
    return torch.cat(outs), torch.cat(lses, 1)
