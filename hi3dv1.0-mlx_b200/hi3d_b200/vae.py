"""Operators of the sparse VAE decoder (``PTv3MeshDecoder``) on B200.

Mirrors the GPU-side pieces of ``SparconvVAEDecoderMLX`` (src/hi3d_mac/mlx_backend/vae.py) and
its helpers:

* :func:`group_stats`, :func:`group_norm_swish`, :func:`conv_gn_swish` -- ``conv(swish(GN(x)))``
  (vae.py:142-192, kernels.py:242-296): statistics by a deterministic two-stage reduction, the
  activated features written once, then the gathered tcgen05 convolution;
* :func:`group_norm_act`, :func:`group_norm_act_backward` -- the norm for training: ragged samples,
  every float type, with its gradient (:mod:`hi3d_b200.training` joins them for autograd);
* :func:`child_neighbour_table` -- the octree child table from the parent table and the
  occupancy masks (sparse.py:46-95), on the GPU;
* :func:`serialization`, :func:`window_index`, :func:`window_attention` -- the serialized
  window attention of the mid attention blocks (vae.py:49-88, :249-266).
"""

from __future__ import annotations

import ctypes
import functools
import math

import numpy as np
import torch

from . import _lib, sparse

PATCH = 48
ORDERS = ("z", "z-trans")


def _groups(c: int) -> int:
    """Groups of ``PointGroupNorm``: 32, or ``c // 4`` for narrow layers (vae.py:150)."""
    return 32 if 4 * 32 <= c else c // 4


def group_stats(x: torch.Tensor, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-channel ``mean`` and ``rsqrt(var + eps)`` of the channel groups (fp32 ``[C]`` each)."""
    _lib.require_cuda(x)
    if x.dtype not in (torch.float16, torch.float32):
        raise ValueError("group_stats takes float16/float32 features")
    x = x.contiguous()
    n, c = x.shape
    mean = torch.empty(c, dtype=torch.float32, device=x.device)
    inv = torch.empty_like(mean)
    lib = _lib.load()
    nb = ctypes.c_int64()
    _lib.check(lib.hi3d_group_norm_stats_workspace_size(n, c, ctypes.byref(nb)), "group_stats", launched=False)
    ws = torch.empty(nb.value, dtype=torch.uint8, device=x.device)
    rc = lib.hi3d_group_norm_stats(x.data_ptr(), n, c, _groups(c), float(eps), mean.data_ptr(), inv.data_ptr(),
                                   ws.data_ptr(), ws.numel(), _lib.dtype_code(x), _lib.stream(x))
    _lib.check(rc, "group_stats")
    return mean, inv


def group_norm_swish(x: torch.Tensor, mean: torch.Tensor, inv: torch.Tensor, weight: torch.Tensor,
                     bias: torch.Tensor, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """``swish((x - mean) * inv * weight + bias)`` in fp32, stored in ``out_dtype``."""
    _lib.require_cuda(x, mean, inv, weight, bias)
    x = x.contiguous()
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    rc = _lib.load().hi3d_group_norm_swish(x.data_ptr(), x.shape[0], x.shape[1], mean.data_ptr(), inv.data_ptr(),
                                           weight.float().contiguous().data_ptr(),
                                           bias.float().contiguous().data_ptr(), out.data_ptr(),
                                           _lib.dtype_code(x), _lib.dtype_code(out), _lib.stream(x))
    _lib.check(rc, "group_norm_swish")
    return out


def conv_gn_swish(x: torch.Tensor, level: sparse.Level, norm_weight: torch.Tensor, norm_bias: torch.Tensor,
                  conv_weight: torch.Tensor, conv_bias: torch.Tensor | None,
                  dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """``conv(swish(GroupNorm(x)))`` (vae.py:166-192): ``conv_weight`` in spconv layout
    ``[Cout, 3, 3, 3, Cin]``; the GEMMs run in ``dtype`` (fp16/bf16)."""
    mean, inv = group_stats(x)
    act = group_norm_swish(x, mean, inv, norm_weight, norm_bias, out_dtype=torch.float16)
    return sparse.conv(act.to(dtype), level.table, conv_weight.to(dtype), conv_bias, n_in=level.n,
                       tap_mask=level.tap_mask)


@functools.lru_cache(maxsize=512)
def _norm_plan(shape, dtype, weight_shape, bias_shape, groups: int, act, eps: float, packed: int | None, devices: tuple):
    """What follows from shapes, types and devices alone, worked out once for each combination: the
    number of samples, the argument structure's sizes, bytes of workspace.  ``packed``: offsets given."""
    if min(devices) < 0:
        raise ValueError("hi3d_b200 operators take CUDA tensors")
    if dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError("group_norm_act takes float16, bfloat16 or float32 features")
    if len(shape) < 2:
        raise ValueError(f"x must be [rows, C] or [samples, ..., C], got {tuple(shape)}")
    if act not in (None, "swish"):
        raise ValueError(f"unknown activation {act!r}")
    if packed is not None and (len(shape) != 2 or packed < 2):
        raise ValueError("offsets are samples + 1 row offsets of packed rows [rows, C]")
    c = shape[-1]
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"{c} channels do not divide into {groups} groups")
    if weight_shape != (c,) or bias_shape != (c,):
        raise ValueError(f"weight and bias must be [{c}]")
    if len(set(devices)) != 1:
        raise ValueError("all tensors must be on the device of x")
    samples = packed - 1 if packed else 1 if len(shape) == 2 else shape[0]
    code = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}[dtype]
    sizes = (math.prod(shape[:-1]), c, samples, groups, int(act is not None), code, eps)
    nb = ctypes.c_int64()
    if samples:
        args = _lib.GroupNormArgs(*[16] * 3, 16 if packed else None, *[16] * 7, *sizes)
        with torch.cuda.device(devices[0]):  # the size follows the device's SM count
            _lib.check(_lib.load().hi3d_group_norm_act_workspace_size(ctypes.byref(args), ctypes.byref(nb)),
                       "group_norm_act", launched=False)
    return samples, sizes, nb.value


def _fp32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.detach().float().contiguous()


def _int32(offsets: torch.Tensor | None) -> torch.Tensor | None:
    if offsets is None or (offsets.dtype is torch.int32 and offsets.is_contiguous() and offsets.dim() == 1):
        return offsets
    if offsets.dim() != 1 or offsets.dtype != torch.int32 and offsets.dtype != torch.int64:
        raise ValueError("offsets must be a one-dimensional int32 (or int64) tensor of samples + 1 row offsets")
    return offsets.to(torch.int32).contiguous()


def group_norm_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, groups: int, eps: float = 1e-6,
                   act: str | None = "swish", offsets: torch.Tensor | None = None,
                   ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(y, mean, rstd)``: ``act(GroupNorm(x))`` over channels-last rows, in fp32, ``y`` rounded once to
    the type of ``x``; ``mean, rstd`` fp32 ``[samples, groups]`` for :func:`group_norm_act_backward`.

    ``x`` is one sample ``[rows, C]``, packed samples ``[rows, C]`` with row ``offsets [samples + 1]``
    (some may be empty; they must cover all rows), or ``[samples, ..., C]``.  ``weight, bias`` ``[C]``.
    """
    offsets = _int32(offsets)
    samples, sizes, nbytes = _norm_plan(
        x.shape, x.dtype, weight.shape, bias.shape, groups, act, float(eps), None if offsets is None else offsets.numel(),
        (x.get_device(), weight.get_device(), bias.get_device(), (x if offsets is None else offsets).get_device()))
    x, weight, bias = x.contiguous(), _fp32(weight), _fp32(bias)
    with _lib.on_device(x):
        y, mean, rstd = torch.empty_like(x), weight.new_empty((samples, groups)), weight.new_empty((samples, groups))
        if samples:
            ws = x.new_empty(nbytes, dtype=torch.uint8)
            args = _lib.GroupNormArgs(x.data_ptr(), weight.data_ptr(), bias.data_ptr(), _lib.ptr(offsets),
                                      mean.data_ptr(), rstd.data_ptr(), y.data_ptr(), None, None, None, None, *sizes)
            rc = _lib.load().hi3d_group_norm_act_fwd(ctypes.byref(args), ws.data_ptr(), nbytes, _lib.stream(x))
            _lib.check(rc, "group_norm_act")
    return y, mean, rstd


def group_norm_act_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                            weight: torch.Tensor, bias: torch.Tensor, act: str | None = "swish",
                            offsets: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dx, dweight, dbias)`` of :func:`group_norm_act`: ``dx`` in the type of ``x``, the others fp32
    ``[C]``, summed over all samples in a fixed order."""
    offsets = _int32(offsets)
    if mean.dim() != 2 or mean.shape != rstd.shape or mean.dtype != torch.float32 or rstd.dtype != torch.float32:
        raise ValueError("mean and rstd must be the float32 [samples, groups] of the forward pass")
    # eps went into rstd: any positive number passes the checks
    samples, sizes, nbytes = _norm_plan(
        x.shape, x.dtype, weight.shape, bias.shape, mean.shape[1], act, 1.0, None if offsets is None else offsets.numel(),
        (x.get_device(), weight.get_device(), bias.get_device(), (x if offsets is None else offsets).get_device(),
         dy.get_device(), mean.get_device(), rstd.get_device()))
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy must be like x {tuple(x.shape)} {x.dtype}, got {tuple(dy.shape)} {dy.dtype}")
    if mean.shape[0] != samples:
        raise ValueError(f"mean and rstd are of {mean.shape[0]} samples, x and offsets of {samples}")
    x, dy, mean, rstd = x.contiguous(), dy.contiguous(), mean.contiguous(), rstd.contiguous()
    weight, bias = _fp32(weight), _fp32(bias)
    with _lib.on_device(x):
        dx, dweight, dbias = torch.empty_like(x), weight.new_empty(x.shape[-1]), weight.new_empty(x.shape[-1])
        if samples:
            ws = x.new_empty(nbytes, dtype=torch.uint8)
            args = _lib.GroupNormArgs(x.data_ptr(), weight.data_ptr(), bias.data_ptr(), _lib.ptr(offsets),
                                      mean.data_ptr(), rstd.data_ptr(), None, dy.data_ptr(), dx.data_ptr(),
                                      dweight.data_ptr(), dbias.data_ptr(), *sizes)
            rc = _lib.load().hi3d_group_norm_act_bwd(ctypes.byref(args), ws.data_ptr(), nbytes, _lib.stream(x))
            _lib.check(rc, "group_norm_act_backward")
        else:
            dweight.zero_()
            dbias.zero_()
    return dx, dweight, dbias


def child_neighbour_table(parent_table: torch.Tensor, child_mask: torch.Tensor):
    """``(table [C, 27], parent [C], slot [C])`` of the kept children (parent-major, slot-minor)
    from the parent table ``[P, 27]`` and the occupancy ``child_mask [P, 8]`` (bool/uint8), as
    ``sparse.child_neighbour_table`` (sparse.py:64-95).  Synchronises once (the child count)."""
    _lib.require_cuda(parent_table, child_mask)
    p = parent_table.shape[0]
    mask = child_mask.to(torch.uint8).contiguous()
    if mask.shape != (p, 8):
        raise ValueError("child_mask must be [P, 8]")
    lib = _lib.load()
    nb = ctypes.c_int64()
    _lib.check(lib.hi3d_child_table_workspace_size(p, ctypes.byref(nb)), "child_table", launched=False)
    ws = torch.empty(nb.value, dtype=torch.uint8, device=mask.device)
    parent = torch.empty(8 * p, dtype=torch.int32, device=mask.device)
    slot = torch.empty_like(parent)
    num = torch.zeros(1, dtype=torch.int32, device=mask.device)
    rc = lib.hi3d_child_structure(mask.data_ptr(), p, parent.data_ptr(), slot.data_ptr(), num.data_ptr(),
                                  ws.data_ptr(), ws.numel(), _lib.stream(mask))
    _lib.check(rc, "child_structure")
    c = int(num.item())
    table = torch.empty((c, 27), dtype=torch.int32, device=mask.device)
    rc = lib.hi3d_child_table(parent_table.contiguous().data_ptr(), p, parent.data_ptr(), slot.data_ptr(), c,
                              ws.data_ptr(), table.data_ptr(), _lib.stream(mask))
    _lib.check(rc, "child_table")
    return table, parent[:c], slot[:c]


def serialization(coords) -> list[tuple[torch.Tensor, torch.Tensor]]:
    """``(perm, inverse)`` of the Morton order and of its x/y-swapped variant (vae.py:58-69)."""
    c = sparse._coords_dev(coords)
    n = c.shape[0]
    depth = int(c.max().item()).bit_length() if n else 0
    lib = _lib.load()
    nb = ctypes.c_int64()
    _lib.check(lib.hi3d_serialize_workspace_size(n, ctypes.byref(nb)), "serialization", launched=False)
    ws = torch.empty(nb.value, dtype=torch.uint8, device=c.device)
    out = []
    for order in ORDERS:
        perm = torch.empty(n, dtype=torch.int32, device=c.device)
        inverse = torch.empty_like(perm)
        rc = lib.hi3d_serialize(c.data_ptr(), n, depth, 1 if order == "z-trans" else 0, perm.data_ptr(),
                                inverse.data_ptr(), ws.data_ptr(), ws.numel(), _lib.stream(c))
        _lib.check(rc, "serialization")
        out.append((perm, inverse))
    return out


def window_index(perm: torch.Tensor, patch: int = PATCH) -> torch.Tensor:
    """Rows in padded window order (vae.py:72-88): windows of ``patch`` serialized points, the
    last one completed with the points before it."""
    n = perm.shape[0]
    if n <= patch:
        return perm
    n_pad = -(-n // patch) * patch
    pad = torch.arange(n_pad, device=perm.device)
    rem = n % patch
    if rem:
        pad[n_pad - patch + rem:] = pad[n_pad - 2 * patch + rem:n_pad - patch].clone()
    return perm[pad].contiguous()


def window_attention(qkv: torch.Tensor, gather: torch.Tensor, heads: int, patch: int = PATCH,
                     scale: float | None = None) -> torch.Tensor:
    """Attention within each serialized window (vae.py:249-266): ``qkv [N, 3 C]`` (layout
    ``[3, heads, D]`` per row), ``gather`` from :func:`window_index`; returns ``[N, C]`` in
    point order."""
    _lib.require_cuda(qkv, gather)
    n, c3 = qkv.shape
    c = c3 // 3
    d = c // heads
    scale = d ** -0.5 if scale is None else scale
    out = torch.empty((n, c), dtype=qkv.dtype, device=qkv.device)
    rc = _lib.load().hi3d_window_attention(qkv.contiguous().data_ptr(), gather.contiguous().data_ptr(), n,
                                           gather.shape[0], patch, heads, d, float(scale), out.data_ptr(),
                                           _lib.dtype_code(qkv), _lib.stream(qkv))
    _lib.check(rc, "window_attention")
    return out
