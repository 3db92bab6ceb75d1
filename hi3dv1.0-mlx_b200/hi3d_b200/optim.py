"""AdamW over many tensors in one launch, states in 32 bits or in 8 (the reference trains nothing).

:func:`adamw_step` is the operator; :class:`AdamW` a ``torch.optim.Optimizer`` around it that owns
the states.  The states of all tensors lie in flat buffers, each tensor at a multiple of
:data:`BLOCK` elements, in order (:func:`state_layout`).  With 8-bit states a block of
:data:`BLOCK` values shares one fp32 scale: ``exp_avg`` holds e4m3 codes of ``m / scale`` and
``exp_avg_sq`` those of ``sqrt(v) / scale``.  16-bit weights are the rounded copy of an fp32 master.
"""

from __future__ import annotations

import ctypes
import itertools

import torch

from . import _lib

BLOCK = 256  # HI3D_ADAMW_BLOCK in include/hi3d_b200.h
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def state_layout(numels: list[int]) -> tuple[list[int], int]:
    """``(offsets, total)``: where each tensor of ``numels`` elements begins in the flat states, and
    their length in elements."""
    at = list(itertools.accumulate((-(-n // BLOCK) * BLOCK for n in numels), initial=0))
    return at[:-1], at[-1]


def _check_state(t: torch.Tensor, name: str, dtype: torch.dtype, total: int, device) -> None:
    if t.dtype != dtype or t.numel() != total or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be {total} contiguous {dtype} elements on {device}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")


def adamw_step(params: list[torch.Tensor], grads: list[torch.Tensor], exp_avg: torch.Tensor,
               exp_avg_sq: torch.Tensor, *, step: int, lr: float, betas: tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 0.01, master: torch.Tensor | None = None,
               scales: torch.Tensor | None = None, grad_scale: torch.Tensor | None = None,
               offsets: list[int] | None = None) -> None:
    """One AdamW step of ``params`` by ``grads``, in place, on the current stream:

    ``p *= 1 - lr * weight_decay; m = b1 m + (1 - b1) g; v = b2 v + (1 - b2) g^2;
    p -= lr / (1 - b1^step) * m / (sqrt(v) / sqrt(1 - b2^step) + eps)`` in fp32: the moments'
    operations are rounded one by one, the update's root and quotient good to 2 units in the last place each.

    Args:
        params, grads: contiguous tensors of one dtype (float32, float16, bfloat16) on one device.
        exp_avg, exp_avg_sq: flat states of ``state_layout``'s total length: float32, or
            float8_e4m3fn with ``scales`` (float32 ``[2, total / BLOCK]``).
        step: the number of this step, from 1.
        master: flat float32 weights, for 16-bit ``params`` only.
        grad_scale: optional float32 scalar on the device that multiplies every gradient (a
            loss scale's inverse, a clipping factor).
        offsets: where each tensor's state begins, if not by ``state_layout`` of these tensors.
    """
    if len(params) != len(grads):
        raise ValueError(f"{len(params)} params, {len(grads)} grads")
    if not params:
        return
    first = params[0]
    _lib.require_cuda(first, exp_avg, exp_avg_sq, master, scales, grad_scale)
    dtype, device = first.dtype, first.device
    if dtype not in DTYPES:
        raise ValueError(f"adamw_step takes float32, float16 or bfloat16 tensors, got {dtype}")
    both = [*params, *grads]
    if ({t.dtype for t in both} != {dtype} or {t.get_device() for t in both} != {first.get_device()}
            or not all(map(torch.Tensor.is_contiguous, both)) or any(p.shape != g.shape for p, g in zip(params, grads))):
        raise ValueError("params and grads must be contiguous, of one dtype and device and alike in pairs")
    numels = [p.numel() for p in params]
    if offsets is None:
        offsets, total = state_layout(numels)
    else:
        total = exp_avg.numel()
        if len(offsets) != len(numels):
            raise ValueError(f"{len(offsets)} offsets for {len(numels)} tensors")
    eight = exp_avg.dtype == torch.float8_e4m3fn
    for t, name in ((exp_avg, "exp_avg"), (exp_avg_sq, "exp_avg_sq")):
        _check_state(t, name, torch.float8_e4m3fn if eight else torch.float32, total, device)
    if (scales is not None) != eight:
        raise ValueError("float8_e4m3fn states need scales, float32 ones have none")
    if eight:
        _check_state(scales, "scales", torch.float32, 2 * (total // BLOCK), device)
    if (master is not None) != (dtype != torch.float32):
        raise ValueError("16-bit params need a master, float32 ones have none")
    if master is not None:
        _check_state(master, "master", torch.float32, total, device)
    if grad_scale is not None:
        _check_state(grad_scale, "grad_scale", torch.float32, 1, device)
    if total == 0:
        return
    n = len(numels)
    args = _lib.AdamWArgs(
        params=(ctypes.c_void_p * n)(*map(torch.Tensor.data_ptr, params)),
        grads=(ctypes.c_void_p * n)(*map(torch.Tensor.data_ptr, grads)),
        numels=(ctypes.c_int64 * n)(*numels), offsets=(ctypes.c_int64 * n)(*offsets), master=_lib.ptr(master),
        exp_avg=exp_avg.data_ptr(), exp_avg_sq=exp_avg_sq.data_ptr(), scales=_lib.ptr(scales),
        grad_scale=_lib.ptr(grad_scale), total=total, step=int(step), lr=float(lr), beta1=float(betas[0]),
        beta2=float(betas[1]), eps=float(eps), weight_decay=float(weight_decay), count=n,
        dtype=_lib.dtype_code(first), state_bits=8 if eight else 32)
    with _lib.on_device(first):
        _lib.check(_lib.load().hi3d_adamw_step(ctypes.byref(args), _lib.stream(first)), "adamw_step")
    _lib.changed(*params, exp_avg, exp_avg_sq, master, scales)


class _Bucket:
    """The flat states of one parameter group's tensors of one dtype and device."""

    def __init__(self, params: list[torch.Tensor], bits: int):
        self.dtype, self.device = dtype, device = params[0].dtype, params[0].device
        self.offsets, total = state_layout([p.numel() for p in params])
        kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
        self.exp_avg = torch.zeros(total, dtype=kind, device=device)
        self.exp_avg_sq = torch.zeros(total, dtype=kind, device=device)
        self.scales = None if bits == 32 else torch.zeros((2, total // BLOCK), device=device)
        self.master = None if dtype == torch.float32 else torch.zeros(total, device=device)
        self.at = {p: i for i, p in enumerate(params)}
        self.shapes = {p: p.shape for p in params}
        self.held: dict[torch.Tensor, dict] = {}  # the views that the optimiser's state has had

    def views(self, p: torch.Tensor) -> dict[str, torch.Tensor]:
        """This tensor's part of each buffer."""
        at, n = self.offsets[self.at[p]], p.numel()
        got = {"exp_avg": self.exp_avg[at:at + n].view(p.shape), "exp_avg_sq": self.exp_avg_sq[at:at + n].view(p.shape)}
        if self.scales is not None:
            got["scales"] = self.scales[:, at // BLOCK:-(-(at + n) // BLOCK)]
        if self.master is not None:
            got["master"] = self.master[at:at + n].view(p.shape)
        return got


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is one launch per parameter group, dtype and step count.

    ``state_bits=8`` holds the moments in 8 bits (2 bytes an element and 8 per 256, against 8 bytes).
    16-bit parameters get an fp32 master, taken from them at their first step and rounded back
    after each: load weights before the first step, or with :meth:`load_state_dict`.  Parameters are
    contiguous.  ``state[p]`` has ``step`` and views of the flat buffers; where a parameter changed its
    type or device, or the optimiser was copied, its state moves into the buffers of its new kind at the
    next step.
    """

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if lr < 0 or eps < 0 or weight_decay < 0 or not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("lr, eps and weight_decay must not be negative, betas lie in [0, 1)")
        self.state_bits = state_bits
        self._home: dict[torch.Tensor, _Bucket] = {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dtype not in DTYPES:
                raise ValueError(f"AdamW takes float32, float16 or bfloat16 parameters, got {p.dtype}")

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "state_bits": self.state_bits}

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        self._home = {}  # the states move into new buffers

    def _housed(self, p: torch.Tensor) -> _Bucket | None:
        """The bucket that was made for ``p`` as it is now."""
        b = self._home.get(p)
        return b if b is not None and b.dtype == p.dtype and b.device == p.device and b.shapes[p] == p.shape else None

    def _bucket(self, index: int, p: torch.Tensor) -> _Bucket:
        """The bucket of ``p`` in group ``index``, made at first use for all the group's tensors of its kind
        that are in none."""
        bucket = self._housed(p)
        if bucket is None:
            _lib.require_cuda(p)
            alike = [q for q in self.param_groups[index]["params"]
                     if q.dtype == p.dtype and q.device == p.device and self._housed(q) is None]
            bucket = _Bucket(alike, self.state_bits)
            self._home.update(dict.fromkeys(alike, bucket))
        return bucket

    def _begin(self, index: int, p: torch.Tensor) -> _Bucket:
        bucket, state = self._bucket(index, p), self.state.get(p)
        if state and p in bucket.held and state["exp_avg"] is bucket.held[p]["exp_avg"]:
            return bucket
        views = bucket.views(p)
        if state:  # of another bucket, or a copy: it moves in
            for name, view in views.items():
                if name in state and state[name].shape != view.shape:
                    raise ValueError(f"{name} of shape {tuple(state[name].shape)} for a parameter of shape {tuple(p.shape)}")
        for name, view in views.items():
            if state and name in state:
                view.copy_(state[name])
            elif name == "master":
                view.copy_(p.detach())
            elif p in bucket.held:  # its state was dropped: nothing of it may remain
                view.zero_()
        bucket.held[p] = views
        self.state[p] = {"step": state["step"] if state else 0, **views}
        return bucket

    @torch.no_grad()
    def step(self, closure=None, grad_scale: torch.Tensor | None = None):
        """One step of every parameter with a gradient.  ``grad_scale``: optional float32 device
        scalar multiplying the gradients."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for index, group in enumerate(self.param_groups):
            calls: dict[tuple, tuple] = {}
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.is_sparse:
                    raise ValueError("AdamW takes dense gradients")
                bucket = self._begin(index, p)
                done = self.state[p]["step"] + 1
                ps, gs, at, _ = calls.setdefault((id(bucket), done), ([], [], [], bucket))
                ps.append(p)
                gs.append(g.contiguous())
                at.append(bucket.offsets[bucket.at[p]])
            for (_, done), (ps, gs, at, bucket) in calls.items():
                adamw_step(ps, gs, bucket.exp_avg, bucket.exp_avg_sq, step=done, lr=group["lr"], betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"], master=bucket.master,
                           scales=bucket.scales, grad_scale=grad_scale, offsets=at)
                for p in ps:
                    self.state[p]["step"] = done
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """Takes over groups and states (of the same ``state_bits`` and parameter dtypes), copied into
        this optimiser's own buffers with their types kept.  A state that does not fit changes nothing; a
        parameter that it does not know starts anew."""
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("state_dict has other parameter groups")
        found = []
        for index, (mine, theirs) in enumerate(zip(self.param_groups, groups)):
            for p, key in zip(mine["params"], theirs["params"]):
                saved = state_dict["state"].get(key)
                if not saved:
                    found.append((p, None, None, None))
                    continue
                bucket = self._bucket(index, p)
                views = bucket.views(p)
                if set(views) != set(saved) - {"step"}:
                    raise ValueError(f"state has {sorted(saved)}, this optimiser keeps {sorted(views)}")
                for name, view in views.items():
                    if saved[name].shape != view.shape or saved[name].dtype != view.dtype:
                        raise ValueError(f"{name} is {tuple(saved[name].shape)} {saved[name].dtype}, expected "
                                         f"{tuple(view.shape)} {view.dtype}")
                found.append((p, bucket, views, saved))
        for p, bucket, views, saved in found:
            if saved is None:
                self.state.pop(p, None)
                continue
            for name, view in views.items():
                view.copy_(saved[name])
            bucket.held[p] = views
            self.state[p] = {"step": int(saved["step"]), **views}
        for mine, theirs in zip(self.param_groups, groups):
            mine.update({k: v for k, v in theirs.items() if k != "params"})
