"""The training operators joined for autograd: attention and group norm with their gradients.

The explicit pairs live beside their forward operators (:mod:`hi3d_b200.attention`,
:mod:`hi3d_b200.vae`); the optimiser step is :mod:`hi3d_b200.optim`.  Gradients are first order
only: a second differentiation raises.  The reference trains nothing
(src/hi3d_mac/torch_backend/attention.py:77-109 serves the upstream model's forward).
"""

from __future__ import annotations

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import attention as _attn
from . import vae as _vae


def _wanted(ctx, grads, first: int = 0):
    return [g if ctx.needs_input_grad[first + i] else None for i, g in enumerate(grads)]


class _Dense(Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, q_layout):
        out, lse = _attn.flash_attention_lse(q, k, v, scale, q_layout)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.scale, ctx.q_layout = scale, q_layout
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, lse = ctx.saved_tensors
        grads = _attn.flash_attention_backward(grad_out, q, k, v, out, lse, ctx.scale, ctx.q_layout)
        return (*_wanted(ctx, grads), None, None)


class _Varlen(Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, max_seqlen_q, scale):
        out, lse = _attn.flash_attn_varlen_lse(q, k, v, cu_q, cu_k, max_seqlen_q, scale)
        ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, lse, cu_q, cu_k = ctx.saved_tensors
        grads = _attn.flash_attn_varlen_backward(grad_out, q, k, v, out, lse, cu_q, cu_k, ctx.scale)
        return (*_wanted(ctx, grads), None, None, None, None)


class _Packed(Function):
    """q, k and v as parts of fused tensors: the gradients are written into fused tensors too."""

    @staticmethod
    def forward(ctx, q, kv, cu_q, cu_k, max_seqlen_q, scale):
        fused = q is None
        parts = kv.unbind(1) if fused else (q, *kv.unbind(1))
        out, lse = _attn.flash_attn_varlen_lse(*parts, cu_q, cu_k, max_seqlen_q, scale)
        ctx.save_for_backward(q, kv, out, lse, cu_q, cu_k)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, kv, out, lse, cu_q, cu_k = ctx.saved_tensors
        dkv = torch.empty(kv.shape, dtype=kv.dtype, device=kv.device)
        dq = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
        parts = kv.unbind(1) if q is None else (q, *kv.unbind(1))
        grads = dkv.unbind(1) if q is None else (dq, *dkv.unbind(1))
        _attn.flash_attn_varlen_backward(grad_out, *parts, out, lse, cu_q, cu_k, ctx.scale, grads=grads)
        return (*_wanted(ctx, (dq, dkv)), None, None, None, None)


class _GroupNorm(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, offsets):
        y, mean, rstd = _vae.group_norm_act(x, weight, bias, groups, eps, act, offsets)
        ctx.save_for_backward(x, weight, bias, mean, rstd, offsets)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd, offsets = ctx.saved_tensors
        dx, dw, db = _vae.group_norm_act_backward(dy, x, mean, rstd, weight, bias, ctx.act, offsets)
        return (*_wanted(ctx, (dx, dw.to(weight.dtype), db.to(bias.dtype))), None, None, None, None)


def flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                    q_layout: str = "bhnd") -> torch.Tensor:
    """Differentiable :func:`hi3d_b200.attention.flash_attention` (grouped key heads allowed)."""
    return _Dense.apply(q, k, v, float(scale), q_layout)


def flash_attn_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                      cu_seqlens_k: torch.Tensor | None, max_seqlen_q: int, scale: float) -> torch.Tensor:
    """Differentiable :func:`hi3d_b200.attention.flash_attn_varlen` (grouped key heads allowed)."""
    return _Varlen.apply(q, k, v, cu_seqlens_q, cu_seqlens_k, int(max_seqlen_q), float(scale))


def flash_attn_varlen_qkvpacked(qkv: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int,
                                scale: float) -> torch.Tensor:
    """Differentiable self-attention of ``qkv [T, 3, H, D]``; the gradient is one tensor like it."""
    if qkv.dim() != 4 or qkv.shape[1] != 3:
        raise ValueError(f"qkv must be [T, 3, H, D], got {tuple(qkv.shape)}")
    return _Packed.apply(None, qkv, cu_seqlens, cu_seqlens, int(max_seqlen), float(scale))


def flash_attn_varlen_kvpacked(q: torch.Tensor, kv: torch.Tensor, cu_seqlens_q: torch.Tensor,
                               cu_seqlens_k: torch.Tensor | None, max_seqlen_q: int, scale: float) -> torch.Tensor:
    """Differentiable cross-attention of ``q [T, H, D]`` over ``kv [S, 2, Hk, D]``."""
    if kv.dim() != 4 or kv.shape[1] != 2:
        raise ValueError(f"kv must be [S, 2, H, D], got {tuple(kv.shape)}")
    return _Packed.apply(q, kv, cu_seqlens_q, cu_seqlens_k, int(max_seqlen_q), float(scale))


def group_norm_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, groups: int, eps: float = 1e-6,
                   act: str | None = "swish", offsets: torch.Tensor | None = None) -> torch.Tensor:
    """Differentiable :func:`hi3d_b200.vae.group_norm_act` (``y`` alone)."""
    return _GroupNorm.apply(x, weight, bias, int(groups), float(eps), act, offsets)
