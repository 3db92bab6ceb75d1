"""Flash attention on the B200 tensor cores (tcgen05 + TMEM, TMA-fed).

:func:`flash_attention` keeps the signature and output layout of
``hi3d_mac.mlx_backend.attention.flash_attention`` (src/hi3d_mac/mlx_backend/attention.py:238-277);
:func:`flash_attn_varlen` is the packed variable-length form the upstream
``flash_attn`` API needs (src/sparc3d/nn/sparse/attention/full_attn.py:56-76).

:func:`flash_attention_lse` / :func:`flash_attention_backward` and their ``flash_attn_varlen_*``
forms are the training pair (the reference runs forward only); :mod:`hi3d_b200.training` joins
them for autograd.

Arithmetic (as the reference kernel, attention.py:19-22): ``S = Q K^T`` in fp32,
online softmax in fp32 in the exp2 domain, ``P`` rounded to the input dtype for
``P V`` which accumulates in fp32, output ``O / l`` rounded once.
"""

from __future__ import annotations

import ctypes
import functools
import itertools
import math
from typing import NamedTuple

import torch

from . import _lib

SUPPORTED_HEAD_DIMS = (64, 96, 128)


def _strides3(t: torch.Tensor, layout: str) -> tuple[int, int, int]:
    """(row, head, batch) element strides of a 4-D tensor in ``bhnd`` / ``bnhd`` layout."""
    s = t.stride()
    if layout == "bhnd":
        return s[2], s[1], s[0]
    return s[1], s[2], s[0]


def _check_inner(t: torch.Tensor, name: str) -> None:
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous head dimension")


class KernelTimer:
    """Optional CUDA-event timing of every attention launch on the launching stream.

    ``start()`` arms it, ``stop()`` synchronises and returns one record per launch
    (``nq``, ``nk`` rows; ``flops`` = 4 * Nq * Nk * H * D for dense launches, None for varlen
    ones; ``ms`` the event-timed duration).
    """

    def __init__(self):
        self.records = None

    def start(self) -> None:
        self.records = []

    def stop(self) -> list[dict]:
        recs, self.records = self.records or [], None
        torch.cuda.synchronize()
        return [dict(r, ms=r.pop("e0").elapsed_time(r.pop("e1"))) for r in recs]


TIMER = KernelTimer()


@functools.lru_cache(maxsize=None)
def _sm_count(device_index: int) -> int:
    return torch.cuda.get_device_properties(device_index).multi_processor_count


# Fixed time of one attention CTA (set-up, Q load and first scores, epilogue) in key blocks:
# ≈ 5670 cycles against ≈ 2525 per 128-key block (cfg1 clock traces).
CTA_OVERHEAD_BLOCKS = 2.25
PARTIAL_FACTOR = 1.2  # measured: the partial kernel + merge against the single pass, same keys


def auto_splits(ctas: int, key_blocks: int, sms: int, max_splits: int = 8) -> int:
    """Key splits per query block for ``ctas`` query-block CTAs over ``key_blocks`` key blocks on
    ``sms`` SMs (one CTA per SM): the s minimising the modelled launch time
    ceil(ctas * s / sms) * (overhead + key_blocks / s), a split launch (the partial kernel, its
    fp32 partials and the merge) charged :data:`PARTIAL_FACTOR` times the single pass, taken only
    when it beats no split by more than 3 %.  Short key ranges (cross-attention) and grids of
    about two waves or more stay unsplit."""
    cost = lambda s: (math.ceil(ctas * s / sms) * (CTA_OVERHEAD_BLOCKS + key_blocks / s)
                      * (PARTIAL_FACTOR if s > 1 else 1.0))
    best, best_t = 1, cost(1)
    for s in range(2, max_splits + 1):
        if key_blocks < 2 * s:
            break
        t = cost(s)
        if t < best_t * 0.97:
            best, best_t = s, t
    return best


def _resolve_splits(k_splits, args: _lib.AttnArgs, dev_tensor: torch.Tensor) -> int:
    if k_splits != "auto":
        return int(k_splits)
    tiles = math.ceil(args.max_seqlen_q / 256)
    bk = 128 if args.head_dim == 64 else 64
    longest_k = args.nk if not args.cu_seqlens_k else args.nk  # packed: bounded by the total
    return auto_splits(tiles * args.num_seqs * args.heads, math.ceil(longest_k / bk), _sm_count(dev_tensor.device.index))


def _launch(args: _lib.AttnArgs, dev_tensor: torch.Tensor, k_splits=1) -> None:
    stream = _lib.stream(dev_tensor)
    splits = _resolve_splits(k_splits, args, dev_tensor)
    rec = TIMER.records is not None
    if rec:
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
    lib = _lib.load()
    if splits > 1:
        nbytes = ctypes.c_int64()
        _lib.check(lib.hi3d_flash_attn_split_workspace_size(ctypes.byref(args), splits, ctypes.byref(nbytes)),
                   "flash_attention split workspace", launched=False)
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev_tensor.device)
        rc = lib.hi3d_flash_attn_fwd_split(ctypes.byref(args), splits, ws.data_ptr(), ws.numel(), stream)
    else:
        rc = lib.hi3d_flash_attn_fwd(ctypes.byref(args), stream)
    _lib.check(rc, "flash_attention")
    if rec:
        e1.record()
        dense = not args.cu_seqlens_q
        flops = 4.0 * args.nq * args.nk * args.heads * args.head_dim * args.num_seqs if dense else None
        TIMER.records.append({"nq": args.nq, "nk": args.nk, "flops": flops, "e0": e0, "e1": e1})


def flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                    q_layout: str = "bhnd", k_splits: int | str = "auto") -> torch.Tensor:
    """``softmax(q k^T * scale) v`` for fp16/bf16 inputs, returned as ``[B, Nq, H * D]``.

    Args:
        q: ``[B, H, Nq, D]`` (``q_layout="bhnd"``) or ``[B, Nq, H, D]`` (``"bnhd"``).
        k, v: ``[B, H, Nk, D]``, or ``[1, H, Nk, D]`` shared by every batch element.
        scale: softmax scale applied to ``q k^T``.
        k_splits: key ranges per query block computed by separate CTAs and merged
            (``hi3d_flash_attn_fwd_split``); ``"auto"`` splits only when the query blocks alone
            leave a partial last wave (e.g. one query shard per GPU).
    """
    _lib.require_cuda(q, k, v)
    if q_layout == "bhnd":
        batch, heads, nq, dim = q.shape
    elif q_layout == "bnhd":
        batch, nq, heads, dim = q.shape
    else:
        raise ValueError(f"unknown q layout {q_layout!r}")
    nk = k.shape[2]
    if (dim not in SUPPORTED_HEAD_DIMS or k.shape[1] != heads or k.shape[3] != dim or k.shape[0] not in (1, batch)
            or v.shape != k.shape):
        raise ValueError(f"unsupported shapes q {tuple(q.shape)} k {tuple(k.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("flash_attention takes float16 (or bfloat16) inputs of one dtype")
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _check_inner(t, n)
    out = torch.empty((batch, nq, heads * dim), dtype=q.dtype, device=q.device)
    if nq == 0 or batch == 0:
        return out
    _launch(_dense_args(q, k, v, out, scale, q_layout), q, k_splits)
    return out


def _dense_args(q, k, v, out, scale: float, q_layout: str) -> _lib.AttnArgs:
    if q_layout == "bhnd":
        batch, heads, nq, dim = q.shape
    else:
        batch, nq, heads, dim = q.shape
    qr, qh, qb = _strides3(q, q_layout)
    kr, kh, kb = _strides3(k, "bhnd")
    vr, vh, vb = _strides3(v, "bhnd")
    if k.shape[0] == 1:
        kb = vb = 0
    return _lib.AttnArgs(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
        q_row=qr, q_head=qh, q_batch=qb, k_row=kr, k_head=kh, k_batch=kb, v_row=vr, v_head=vh, v_batch=vb,
        o_row=heads * dim, o_head=dim, o_batch=nq * heads * dim,
        cu_seqlens_q=None, cu_seqlens_k=None, nq=nq, nk=k.shape[2], max_seqlen_q=nq,
        num_seqs=batch, heads=heads, head_dim=dim, dtype=_lib.dtype_code(q), scale=float(scale))


def auto_key_splits(q_rows: int, k_rows: int, heads: int, head_dim: int, batch: int = 1, device=None) -> int:
    """The key splits :func:`flash_attention` picks with ``k_splits="auto"`` for these sizes."""
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    bk = 128 if head_dim == 64 else 64
    return auto_splits(math.ceil(q_rows / 256) * batch * heads, math.ceil(k_rows / bk), _sm_count(dev.index))


class AttentionParts:
    """Attention of one set of queries over several disjoint key sets, combined exactly by their
    log-sum-exp weights: :meth:`add` one key set at a time (``hi3d_flash_attn_fwd_partial``), then
    :meth:`merge` (``hi3d_flash_attn_merge``), or finish with :meth:`add_final`, which merges in
    the last launch's epilogue.  For key sets that arrive at different times; the sharded block
    gathers all keys first and attends them in one pass, which measured faster.  Queries and keys as in
    :func:`flash_attention`; ``slots`` bounds the total key splits of all ``add`` calls."""

    def __init__(self, q: torch.Tensor, scale: float, slots: int, q_layout: str = "bhnd"):
        _lib.require_cuda(q)
        if q_layout not in ("bhnd", "bnhd"):
            raise ValueError(f"unknown q layout {q_layout!r}")
        _check_inner(q, "q")
        self.q, self.scale, self.layout = q, float(scale), q_layout
        if q_layout == "bhnd":
            self.batch, self.heads, self.nq, self.dim = q.shape
        else:
            self.batch, self.nq, self.heads, self.dim = q.shape
        rows = self.batch * self.nq
        self.part_o = torch.empty((slots, rows, self.heads, self.dim), dtype=torch.float32, device=q.device)
        self.part_lse = torch.empty((slots, rows, self.heads), dtype=torch.float32, device=q.device)
        self.slots, self.used = slots, 0

    def add(self, k: torch.Tensor, v: torch.Tensor, k_splits: int | str = "auto") -> None:
        _lib.require_cuda(k, v)
        if k.shape[1] != self.heads or k.shape[3] != self.dim or v.shape != k.shape or k.dtype != self.q.dtype:
            raise ValueError(f"keys {tuple(k.shape)} do not match the queries")
        for t, n in ((k, "k"), (v, "v")):
            _check_inner(t, n)
        if k.shape[2] == 0 or self.nq == 0 or self.batch == 0:
            return
        args = _dense_args(self.q, k, v, self.part_o, self.scale, self.layout)
        splits = _resolve_splits(k_splits, args, self.q)
        if self.used + splits > self.slots:
            raise ValueError(f"{self.used + splits} key splits exceed the {self.slots} partial slots")
        rec = TIMER.records is not None
        if rec:
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record()
        rc = _lib.load().hi3d_flash_attn_fwd_partial(ctypes.byref(args), splits, self.used, self.part_o.data_ptr(),
                                                     self.part_lse.data_ptr(), self.batch * self.nq,
                                                     _lib.stream(self.q))
        _lib.check(rc, "flash_attention partial")
        if rec:
            e1.record()
            flops = 4.0 * args.nq * args.nk * args.heads * args.head_dim * args.num_seqs
            TIMER.records.append({"nq": args.nq, "nk": args.nk, "flops": flops, "e0": e0, "e1": e1, "part": True})
        self.used += splits

    def add_final(self, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """The last key set in one pass, merged with the partials added so far inside the
        attention kernel's epilogue (``hi3d_flash_attn_fwd_partial_merge``); returns the
        ``[B, Nq, H * D]`` output that :meth:`merge` would return after ``add(k, v, 1)``."""
        _lib.require_cuda(k, v)
        if k.shape[1] != self.heads or k.shape[3] != self.dim or v.shape != k.shape or k.dtype != self.q.dtype:
            raise ValueError(f"keys {tuple(k.shape)} do not match the queries")
        for t, n in ((k, "k"), (v, "v")):
            _check_inner(t, n)
        if k.shape[2] == 0:
            return self.merge()
        out = torch.empty((self.batch, self.nq, self.heads * self.dim), dtype=self.q.dtype, device=self.q.device)
        if self.nq == 0 or self.batch == 0:
            return out
        args = _dense_args(self.q, k, v, out, self.scale, self.layout)
        rec = TIMER.records is not None
        if rec:
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record()
        rc = _lib.load().hi3d_flash_attn_fwd_partial_merge(ctypes.byref(args), self.used, self.part_o.data_ptr(),
                                                           self.part_lse.data_ptr(), self.batch * self.nq,
                                                           _lib.stream(self.q))
        _lib.check(rc, "flash_attention partial merge")
        if rec:
            e1.record()
            flops = 4.0 * args.nq * args.nk * args.heads * args.head_dim * args.num_seqs
            TIMER.records.append({"nq": args.nq, "nk": args.nk, "flops": flops, "e0": e0, "e1": e1, "part": True})
        return out

    def merge(self) -> torch.Tensor:
        """``[B, Nq, H * D]`` from all key sets added so far."""
        out = torch.empty((self.batch, self.nq, self.heads * self.dim), dtype=self.q.dtype, device=self.q.device)
        if self.used == 0 or self.nq == 0 or self.batch == 0:
            return out
        args = _dense_args(self.q, self.q if self.layout == "bhnd" else self.q.transpose(1, 2),
                           self.q if self.layout == "bhnd" else self.q.transpose(1, 2), out, self.scale, self.layout)
        rc = _lib.load().hi3d_flash_attn_merge(ctypes.byref(args), self.used, self.part_o.data_ptr(),
                                               self.part_lse.data_ptr(), _lib.stream(self.q))
        _lib.check(rc, "flash_attention merge")
        return out


def flash_attn_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                      cu_seqlens_k: torch.Tensor | None, max_seqlen_q: int, scale: float,
                      out: torch.Tensor | None = None, k_splits: int | str = "auto") -> torch.Tensor:
    """Packed variable-length attention: ``q [Tq, H, D]``, ``k, v [Tk, H, D]`` (any row
    stride, contiguous head dim), ``cu_seqlens_*`` int32 ``[num_seqs + 1]`` on the device.
    ``cu_seqlens_k=None`` shares all ``Tk`` keys with every sequence.  Returns ``[Tq, H, D]``.
    ``k_splits`` as in :func:`flash_attention`.
    """
    _lib.require_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k)
    tq, heads, dim = q.shape
    tk = k.shape[0]
    if dim not in SUPPORTED_HEAD_DIMS or k.shape[1:] != (heads, dim) or v.shape[1:] != (heads, dim):
        raise ValueError(f"unsupported shapes q {tuple(q.shape)} k {tuple(k.shape)} v {tuple(v.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("flash attention takes float16 or bfloat16 inputs of one dtype")
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _check_inner(t, n)
    cu_q = cu_seqlens_q.to(torch.int32).contiguous()
    cu_k = None if cu_seqlens_k is None else cu_seqlens_k.to(torch.int32).contiguous()
    num_seqs = cu_q.numel() - 1
    if cu_k is not None and cu_k.numel() != cu_q.numel():
        raise ValueError("cu_seqlens_q and cu_seqlens_k must have the same length")
    if out is None:
        out = torch.empty((tq, heads, dim), dtype=q.dtype, device=q.device)
    if tq == 0 or num_seqs <= 0:
        return out
    args = _lib.AttnArgs(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
        q_row=q.stride(0), q_head=q.stride(1), q_batch=0, k_row=k.stride(0), k_head=k.stride(1), k_batch=0,
        v_row=v.stride(0), v_head=v.stride(1), v_batch=0,
        o_row=out.stride(0), o_head=out.stride(1), o_batch=0,
        cu_seqlens_q=cu_q.data_ptr(), cu_seqlens_k=None if cu_k is None else cu_k.data_ptr(),
        nq=tq, nk=tk, max_seqlen_q=int(max_seqlen_q), num_seqs=num_seqs, heads=heads, head_dim=dim,
        dtype=_lib.dtype_code(q), scale=float(scale))
    _launch(args, q, k_splits)
    return out


# ---------------------------------------------------------------------------
# training: the forward pass with its log-sum-exp, and the gradients
# ---------------------------------------------------------------------------
# A call's checks and strides depend on shapes, strides, types and devices alone, so they are worked
# out once for each combination (a plan) and kept; addresses are looked at on every call.
def _lies(shape, stride) -> bool:
    """Whether the kernels' 16-byte loads and TMA boxes can address these strides."""
    return stride[-1] == 1 and all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(shape[:-1], stride[:-1]))


def _fit(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself, or a contiguous copy where its strides or address do not fit the kernels
    (an expanded gradient, an odd slice)."""
    if t.data_ptr() % 16 == 0 and _lies(t.shape, t.stride()):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _steps(shape, stride, row: int, head: int, batch: int | None = None) -> tuple[int, int, int]:
    """Element strides of these axes.  An axis of one element may have any stride, which the kernels
    would refuse: a row or head then steps by one head, a batch by 0 (one set for every sequence)."""
    return (stride[row] if shape[row] != 1 else shape[-1], stride[head] if shape[head] != 1 else shape[-1],
            0 if batch is None or shape[batch] == 1 else stride[batch])


def _contiguous(shape) -> tuple[int, ...]:
    return tuple(itertools.accumulate(reversed(shape[1:]), lambda a, b: a * max(b, 1), initial=1))[::-1]


class _Plan(NamedTuple):
    batch: int      # dense: sequences; packed: 1
    heads: int
    nq: int         # rows of a sequence, packed: of all
    nk: int
    kv_heads: int
    dim: int
    dtype: int
    q_axes: tuple   # (row, head[, batch]) of q and dq
    k_axes: tuple
    steps: tuple    # nine strides of q, k, v
    fits: bool
    out_shape: tuple
    lse_shape: tuple
    out_steps: tuple


@functools.lru_cache(maxsize=512)
def _plan(layout: str, qs, qt, ks, kt, vs, vt, types: tuple, devices: tuple) -> _Plan:
    """Checks and strides of queries, keys and values; layout ``bhnd``, ``bnhd`` or ``packed``."""
    if min(devices) < 0:
        raise ValueError("hi3d_b200 operators take CUDA tensors")
    if layout not in ("bhnd", "bnhd", "packed"):
        raise ValueError(f"unknown q layout {layout!r}")
    rank = 3 if layout == "packed" else 4
    if len(qs) != rank or len(ks) != rank:
        raise ValueError(f"unsupported shapes q {tuple(qs)} k {tuple(ks)} v {tuple(vs)}")
    q_axes = {"bhnd": (2, 1, 0), "bnhd": (1, 2, 0), "packed": (0, 1)}[layout]
    k_axes = (0, 1) if layout == "packed" else (2, 1, 0)
    nq, heads, batch = qs[q_axes[0]], qs[q_axes[1]], 1 if rank == 3 else qs[0]
    nk, kv_heads, dim = ks[k_axes[0]], ks[k_axes[1]], qs[-1]
    if dim not in SUPPORTED_HEAD_DIMS:
        raise NotImplementedError(f"head_dim {dim} not supported {SUPPORTED_HEAD_DIMS}")
    if (ks != vs or ks[-1] != dim or (rank == 4 and ks[0] not in (1, batch)) or kv_heads < 1 or heads < 1
            or heads % kv_heads):
        raise ValueError(f"unsupported shapes q {tuple(qs)} k {tuple(ks)} v {tuple(vs)}")
    if types[0] not in (torch.float16, torch.bfloat16) or len(set(types)) != 1:
        raise ValueError("flash attention takes float16 or bfloat16 inputs of one dtype")
    if len(set(devices)) != 1:
        raise ValueError("q, k and v must be on one device")
    return _Plan(batch, heads, nq, nk, kv_heads, dim, _lib.F16 if types[0] == torch.float16 else _lib.BF16, q_axes,
                 k_axes, (*_steps(qs, qt, *q_axes), *_steps(ks, kt, *k_axes), *_steps(vs, vt, *k_axes)),
                 _lies(qs, qt) and _lies(ks, kt) and _lies(vs, vt),
                 (nq, heads, dim) if rank == 3 else (batch, nq, heads * dim),
                 (heads, nq) if rank == 3 else (batch, heads, nq),
                 (heads * dim, dim, 0 if rank == 3 else nq * heads * dim))


def _planned(layout: str, q, k, v):
    """The plan of these tensors, and they or copies that fit the kernels."""
    for _ in range(2):
        p = _plan(layout, q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), (q.dtype, k.dtype, v.dtype),
                  (q.get_device(), k.get_device(), v.get_device()))
        if p.nq == 0 or p.nk == 0 or p.batch == 0 or (
                p.fits and not (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15):
            break
        q, k, v = _fit(q), _fit(k), _fit(v)
    return p, q, k, v


def _scale(scale) -> float:
    scale = float(scale)
    if not 0.0 <= scale < math.inf:
        raise ValueError(f"scale must be finite and not negative, got {scale}")
    return scale


def _cu(cu: torch.Tensor | None, like: torch.Tensor, name: str) -> torch.Tensor | None:
    if cu is None:
        return None
    if cu.dim() != 1 or cu.numel() < 1 or cu.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be a one-dimensional int32 (or int64) tensor of num_seqs + 1 offsets")
    if cu.get_device() != like.get_device():
        raise ValueError(f"{name} must be on the device of q")
    return cu if cu.dtype is torch.int32 and cu.is_contiguous() else cu.to(torch.int32).contiguous()


def _offsets(cu_seqlens_q, cu_seqlens_k, q):
    cu_q, cu_k = _cu(cu_seqlens_q, q, "cu_seqlens_q"), _cu(cu_seqlens_k, q, "cu_seqlens_k")
    if cu_k is not None and cu_k.numel() != cu_q.numel():
        raise ValueError("cu_seqlens_q and cu_seqlens_k must have the same length")
    return cu_q, cu_k


_cached_splits = functools.lru_cache(maxsize=512)(auto_splits)


def _forward_lse(p: _Plan, q, k, v, cu_q, cu_k, num_seqs: int, longest: int, scale: float, k_splits):
    with _lib.on_device(q):
        if p.nk == 0:
            return q.new_zeros(p.out_shape), torch.full(p.lse_shape, -math.inf, device=q.device)
        out, lse = q.new_empty(p.out_shape), q.new_empty(p.lse_shape, dtype=torch.float32)
        if p.nq == 0 or num_seqs == 0:
            return out, lse
        args = _lib.AttnArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), *p.steps, *p.out_steps,
                             _lib.ptr(cu_q), _lib.ptr(cu_k), p.nq, p.nk, longest, num_seqs, p.heads, p.dim, p.dtype,
                             scale)
        if k_splits == "auto":
            k_splits = _cached_splits(math.ceil(longest / 256) * num_seqs * p.heads,
                                      math.ceil(p.nk / (128 if p.dim == 64 else 64)), _sm_count(q.get_device()))
        lib, ws, nbytes = _lib.load(), None, ctypes.c_int64()
        if k_splits > 1:
            _lib.check(lib.hi3d_flash_attn_split_workspace_size(ctypes.byref(args), k_splits, ctypes.byref(nbytes)),
                       "flash_attention split workspace", launched=False)
            ws = q.new_empty(nbytes.value, dtype=torch.uint8)
        rc = lib.hi3d_flash_attn_fwd_lse(ctypes.byref(args), p.kv_heads, lse.data_ptr(), int(k_splits), _lib.ptr(ws),
                                         nbytes.value, _lib.stream(q))
        _lib.check(rc, "flash_attention_lse")
    return out, lse


def flash_attention_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, q_layout: str = "bhnd",
                        k_splits: int | str = "auto") -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`flash_attention` for training: ``(out [B, Nq, H * D], lse [B, H, Nq])`` with the fp32
    log-sum-exp of each row's scaled scores, which :func:`flash_attention_backward` takes.

    ``k, v`` ``[B or 1, Hk, Nk, D]`` with ``Hk`` dividing ``H``: query head ``h`` reads key head
    ``h // (H // Hk)``.  Without keys (``Nk = 0``) the output is 0 and ``lse`` is ``-inf``.
    """
    if q_layout == "packed":
        raise ValueError(f"unknown q layout {q_layout!r}")
    p, q, k, v = _planned(q_layout, q, k, v)
    return _forward_lse(p, q, k, v, None, None, p.batch, p.nq, _scale(scale), k_splits)


def flash_attn_varlen_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                          cu_seqlens_k: torch.Tensor | None, max_seqlen_q: int, scale: float,
                          k_splits: int | str = "auto") -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`flash_attn_varlen` for training: ``(out [Tq, H, D], lse [H, Tq])``.

    ``k, v`` ``[Tk, Hk, D]`` with ``Hk`` dividing ``H``.  A sequence without keys gets an output of 0
    and ``lse = -inf``.  Sequences never see each other's rows, NaN and infinities included.  The
    offsets must cover all rows of ``q``, and no sequence may be longer than ``max_seqlen_q``.
    """
    p, q, k, v = _planned("packed", q, k, v)
    cu_q, cu_k = _offsets(cu_seqlens_q, cu_seqlens_k, q)
    num_seqs = cu_q.numel() - 1
    if int(max_seqlen_q) < 1 and p.nq and num_seqs:
        raise ValueError("max_seqlen_q must be at least the longest query sequence")
    return _forward_lse(p, q, k, v, cu_q, cu_k, num_seqs, min(int(max_seqlen_q), p.nq), _scale(scale), k_splits)


@functools.lru_cache(maxsize=512)
def _saved_plan(p: _Plan, os, ot, gs, gt, ls, types: tuple, devices: tuple) -> tuple:
    """Checks of what the backward pass is given beside q, k, v, and the strides of out and its
    gradient, or None where a copy has to be made."""
    for name, shape, kind, device in zip(("out", "grad_out"), (os, gs), types, devices):
        if shape != p.out_shape or kind != types[3] or device != devices[3]:
            raise ValueError(f"{name} must be {p.out_shape} in the dtype and on the device of q, got {tuple(shape)}")
    if ls != p.lse_shape or types[2] != torch.float32 or devices[2] != devices[3]:
        raise ValueError(f"lse must be the float32 {p.lse_shape} of the forward pass, got {tuple(ls)}")
    steps = []
    for shape, stride in ((os, ot), (gs, gt)):
        if len(shape) == 3 and len(p.q_axes) == 3:  # [B, Nq, H * D] as [B, Nq, H, D]
            shape, stride = (*shape[:2], p.heads, p.dim), (*stride[:2], p.dim * stride[2], stride[2])
        axes = (0, 1) if len(shape) == 3 else (1, 2, 0)
        steps.append(_steps(shape, stride, *axes) if _lies(shape, stride) else None)
    return tuple(steps)


@functools.lru_cache(maxsize=512)
def _backward_plan(p: _Plan, qs, ks, steps: tuple, packed_k: bool, num_seqs: int, scale: float, device: int) -> tuple:
    """(the argument structure's strides with contiguous gradients, its sizes, bytes of workspace)."""
    dq, dk = _steps(qs, _contiguous(qs), *p.q_axes), _steps(ks, _contiguous(ks), *p.k_axes)
    sizes = (p.nq, p.nk, num_seqs, p.heads, p.kv_heads, p.dim, p.dtype, scale)
    packed = len(p.q_axes) == 2
    # only the presence of pointers counts for the workspace
    args = _lib.AttnBwdArgs(*[16] * 9, *p.steps, *steps, *dq, *dk, *dk, 16 if packed else None,
                            16 if packed_k else None, *sizes)
    nbytes = ctypes.c_int64()
    _lib.check(_lib.load().hi3d_flash_attn_bwd_workspace_size(ctypes.byref(args), ctypes.byref(nbytes)),
               "flash_attention_backward workspace", launched=False)
    return (*p.steps, *steps, *dq, *dk, *dk), sizes, nbytes.value


def _given(grads, like, p: _Plan) -> tuple[list, tuple]:
    """The caller's gradient tensors, checked, with new ones for None, and their strides."""
    got, steps = [], []
    for name, g, t, axes in zip(("dq", "dk", "dv"), grads, like, (p.q_axes, p.k_axes, p.k_axes)):
        if g is None:
            g = t.new_empty(t.shape)
        elif (g.shape != t.shape or g.dtype != t.dtype or g.device != t.device or g.data_ptr() % 16
              or not _lies(g.shape, g.stride())):
            raise ValueError(f"{name} must have the shape, dtype and device of its input, rows contiguous over the "
                             "head dimension and 16-byte aligned")
        got.append(g)
        steps += _steps(g.shape, g.stride(), *axes)
    return got, tuple(steps)


def _backward(p: _Plan, grad_out, q, k, v, out, lse, cu_q, cu_k, num_seqs: int, scale: float, grads):
    for _ in range(2):
        steps = _saved_plan(p, out.shape, out.stride(), grad_out.shape, grad_out.stride(), lse.shape,
                            (out.dtype, grad_out.dtype, lse.dtype, q.dtype),
                            (out.get_device(), grad_out.get_device(), lse.get_device(), q.get_device()))
        if None not in steps and not (out.data_ptr() | grad_out.data_ptr()) & 15:
            break
        if p.nq == 0 or p.nk == 0 or p.batch == 0 or num_seqs == 0:
            break
        out, grad_out = _fit(out), _fit(grad_out)
    with _lib.on_device(q):
        if grads is None:
            dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
            given = None
        else:
            (dq, dk, dv), given = _given(grads, (q, k, v), p)
            _lib.changed(*grads)
        if p.nq == 0 or p.nk == 0 or p.batch == 0 or num_seqs == 0:
            for t in (dq, dk, dv):
                t.zero_()
            return dq, dk, dv
        strides, sizes, nbytes = _backward_plan(p, q.shape, k.shape, steps[0] + steps[1], cu_k is not None, num_seqs,
                                                scale, q.get_device())
        if given is not None:
            strides = strides[:15] + given
        lse = lse.contiguous()
        args = _lib.AttnBwdArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), grad_out.data_ptr(),
                                lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *strides, _lib.ptr(cu_q),
                                _lib.ptr(cu_k), *sizes)
        ws = q.new_empty(nbytes, dtype=torch.uint8)
        rc = _lib.load().hi3d_flash_attn_bwd(ctypes.byref(args), ws.data_ptr(), nbytes, _lib.stream(q))
        _lib.check(rc, "flash_attention_backward")
    return dq, dk, dv


def flash_attention_backward(grad_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                             out: torch.Tensor, lse: torch.Tensor, scale: float, q_layout: str = "bhnd",
                             grads: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dq, dk, dv)`` of :func:`flash_attention_lse` in the shapes of ``q, k, v``.

    ``dk, dv`` sum over the query heads of a group, and over the batch where the keys are shared.
    Probabilities are recomputed from ``lse``; P and dS are rounded to the input dtype for the
    products, sums are fp32 in a fixed order (the same bits on every run), each gradient is rounded
    once.  ``grads``: optional ``(dq, dk, dv)`` tensors to write, e.g. views of one fused gradient
    (None entries are allocated).
    """
    if q_layout == "packed":
        raise ValueError(f"unknown q layout {q_layout!r}")
    p, q, k, v = _planned(q_layout, q, k, v)
    return _backward(p, grad_out, q, k, v, out, lse, None, None, p.batch, _scale(scale), grads)


def flash_attn_varlen_backward(grad_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                               out: torch.Tensor, lse: torch.Tensor, cu_seqlens_q: torch.Tensor,
                               cu_seqlens_k: torch.Tensor | None, scale: float,
                               grads: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dq, dk, dv)`` of :func:`flash_attn_varlen_lse` in the shapes of ``q, k, v``, as
    :func:`flash_attention_backward`; with ``cu_seqlens_k=None`` ``dk, dv`` sum over all sequences.
    No longest length is needed.  Gradient rows outside the offsets are not written."""
    p, q, k, v = _planned("packed", q, k, v)
    cu_q, cu_k = _offsets(cu_seqlens_q, cu_seqlens_k, q)
    return _backward(p, grad_out, q, k, v, out, lse, cu_q, cu_k, cu_q.numel() - 1, _scale(scale), grads)
