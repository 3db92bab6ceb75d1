"""``flash_attn`` varlen functions backed by the B200 tcgen05 attention kernel.

Same signatures as the functions the upstream code calls
(src/sparc3d/nn/sparse/attention/full_attn.py:56-76) and as the reference's CPU shim
(src/hi3d_mac/torch_backend/attention.py:77-109), including its errors for causal or
dropout attention.  Inputs are fp16/bf16 CUDA tensors, as for flash-attn itself.  Where a gradient is
wanted they run the training pair (:mod:`hi3d_b200.training`): attention and torch's own layers of the
upstream model train; its sparse convolutions (sparse_conv.py) run forward only and say so in ``backward``.
"""

from __future__ import annotations

import torch

from .. import attention as _attn
from .. import training as _train


def _wants_grad(*ts: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in ts)


def flash_attn_varlen_qkvpacked_func(qkv: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int,
                                     dropout_p: float = 0.0, softmax_scale: float | None = None,
                                     causal: bool = False, **_: object) -> torch.Tensor:
    """Self-attention over packed ``[T, 3, H, D]`` sequences; returns ``[T, H, D]``."""
    if causal or dropout_p:
        raise NotImplementedError("causal or dropout attention is not used by Hi3D")
    scale = qkv.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale
    if scale < 0:
        return flash_attn_varlen_kvpacked_func(qkv[:, 0], qkv[:, 1:], cu_seqlens.to(qkv.device),
                                               cu_seqlens.to(qkv.device), max_seqlen, max_seqlen, softmax_scale=scale)
    if _wants_grad(qkv):
        return _train.flash_attn_varlen_qkvpacked(qkv, cu_seqlens.to(qkv.device), int(max_seqlen), scale)
    q, k, v = qkv.unbind(1)
    return _attn.flash_attn_varlen(q, k, v, cu_seqlens, cu_seqlens, int(max_seqlen), scale)


def flash_attn_varlen_kvpacked_func(q: torch.Tensor, kv: torch.Tensor, cu_seqlens_q: torch.Tensor,
                                    cu_seqlens_k: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int,
                                    dropout_p: float = 0.0, softmax_scale: float | None = None,
                                    causal: bool = False, **_: object) -> torch.Tensor:
    """Cross-attention of packed queries ``[T, H, D]`` over packed ``[S, 2, H, D]``."""
    if causal or dropout_p:
        raise NotImplementedError("causal or dropout attention is not used by Hi3D")
    scale = q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale
    if scale < 0:  # the kernels' masked scores are -inf and have to stay it
        q, scale = -q, -scale
    if _wants_grad(q, kv):
        return _train.flash_attn_varlen_kvpacked(q, kv, cu_seqlens_q.to(q.device), cu_seqlens_k.to(q.device),
                                                 int(max_seqlen_q), scale)
    k, v = kv.unbind(1)
    return _attn.flash_attn_varlen(q, k, v, cu_seqlens_q.to(q.device), cu_seqlens_k.to(q.device),
                                   int(max_seqlen_q), scale)
