"""Differentiable forms of the operators for training on packed images and clips (ops.layer_norm_fwd, ops.rope_axes, ops.attn_packed): torch.autograd
functions around the operators and their gradients, for models that are fine-tuned with autograd.

They run eagerly.  Inside a CUDA graph capture they refuse to take part in autograd (KfError): a gradient that is accumulated into a leaf which an
eager graph also holds would make the capturing stream wait for one that is not captured, and torch ends the process there.  The operators
themselves can be captured in both directions; call those."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import KfError


def _capturing(t: torch.Tensor) -> bool:
    """does the stream capture that an operator on t launches on: the current one of its device"""
    if t.device.index == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(t.device):
        return torch.cuda.is_current_stream_capturing()


def _eager_backward(t: torch.Tensor) -> None:
    if _capturing(t):
        raise KfError("grad: no autograd inside a CUDA graph capture; capture the operators of ops (forward and gradient) instead")


def _eager(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors) and tensors[0].device.type == "cuda":
        _eager_backward(tensors[0])


def _rows(g: torch.Tensor, align: int = 1) -> torch.Tensor:
    """a gradient as the kernels take it: contiguous, at a multiple of `align` bytes (autograd hands on expanded and permuted ones, and views of others at any offset)"""
    g = g if g.is_contiguous() else g.contiguous()
    return g if g.data_ptr() % align == 0 else g.clone()


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps, dtype):
        y, mean, rstd = ops.layer_norm_fwd(x, w, b, eps, dtype)
        ctx.save_for_backward(x, w, mean, rstd)
        ctx.bias = b is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, mean, rstd = ctx.saved_tensors
        _eager_backward(x)
        dx, dw, db = ops.layer_norm_bwd(_rows(dy), x, w, mean, rstd, bias=ctx.bias, affine=any(ctx.needs_input_grad[1:3]))
        return dx, dw, db, None, None


class _RopeAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, table):
        ctx.save_for_backward(pos)
        ctx.table = table
        return ops.rope_axes(x, pos, table)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _eager_backward(dy)
        return ops.rope_axes(_rows(dy, 2 * dy.element_size() if ctx.table.interleaved else 1), *ctx.saved_tensors, ctx.table, inverse=True), None, None


class _AttnPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, plan, scale, cap, slopes):
        out, lse = ops.attn_packed(q, k, v, plan, scale=scale, cap=cap, slopes=slopes)
        ctx.save_for_backward(q, k, v, out, lse, slopes)
        ctx.how = (plan, scale, cap)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, slopes = ctx.saved_tensors
        plan, scale, cap = ctx.how
        _eager_backward(q)
        return (*ops.attn_packed_bwd(_rows(dout, 16), q, k, v, out, lse, plan, scale=scale, cap=cap, slopes=slopes, keys=any(ctx.needs_input_grad[1:3])), None, None, None, None)


def layer_norm(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor], eps: float, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """ops.layer_norm_fwd's y, differentiable in x, w and b."""
    _eager(x, w, b)
    return _LayerNorm.apply(x, w, b, eps, dtype)


def rope_axes(x: torch.Tensor, pos: torch.Tensor, table: ops.RopeTable) -> torch.Tensor:
    """ops.rope_axes, differentiable in x."""
    _eager(x)
    return _RopeAxes.apply(x, pos, table)


def attn_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: ops.AttnPlan, *, scale: Optional[float] = None, cap: float = 0.0,
                slopes: Optional[torch.Tensor] = None) -> torch.Tensor:
    """ops.attn_packed's out, differentiable in q, k and v.  slopes are constants: one that requires a gradient is refused."""
    _eager(q, k, v)
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise KfError("grad.attn_packed: slopes have no gradient")
    return _AttnPacked.apply(q, k, v, plan, scale, cap, slopes)
