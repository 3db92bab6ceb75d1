"""The optimiser's book-keeping on the CPU: which state a parameter steps on.  The step itself is a plain
AdamW here (on the GPU: test_adamw_gpu.py); the comparisons are bit for bit."""

from __future__ import annotations

import pytest
import torch

from hi3d_b200 import _lib, optim


def _plain_step(params, grads, exp_avg, exp_avg_sq, *, step, lr, betas, eps, weight_decay, master, scales, grad_scale,
                offsets):
    for p, g, at in zip(params, grads, offsets):
        part = lambda t: t[at:at + p.numel()].view(p.shape)  # noqa: E731
        g = g.float()
        if scales is not None:  # 8 bits: only that a step leaves something behind
            part(exp_avg).copy_(g)
            part(exp_avg_sq).copy_(g)
            scales[:, at // optim.BLOCK:-(-(at + p.numel()) // optim.BLOCK)] += 1
            continue
        m, v = part(exp_avg).lerp_(g, 1 - betas[0]), part(exp_avg_sq).lerp_(g * g, 1 - betas[1])
        w = p if master is None else part(master)
        w.mul_(1 - lr * weight_decay)
        w.sub_(lr / (1 - betas[0] ** step) * m / (v.sqrt() * (1 - betas[1] ** step) ** -0.5 + eps))
        if master is not None:
            p.copy_(w)


@pytest.fixture(autouse=True)
def _on_the_cpu(monkeypatch):
    monkeypatch.setattr(optim, "adamw_step", _plain_step)
    monkeypatch.setattr(_lib, "require_cuda", lambda *ts: None)


def _params(dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype)) for s in ((300,), (5, 7), (256,))]


def _steps(opt, ps, seeds):
    for seed in seeds:
        g = torch.Generator().manual_seed(100 + seed)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(p.dtype)
        opt.step()


def _equal(ps, qs):
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("how", ["load", "clear", "partial"])
def test_a_parameter_without_state_starts_anew(dtype, how):
    """After a load of a state that does not know it, or after the state was cleared, a parameter steps as in
    a new optimiser: zero moments, a master from the weights as they are."""
    ps = _params(dtype)
    opt = optim.AdamW(ps, lr=1e-2)
    _steps(opt, ps, range(3))
    if how == "load":
        opt.load_state_dict(optim.AdamW(_params(dtype), lr=1e-2).state_dict())
    elif how == "partial":
        saved = opt.state_dict()
        del saved["state"][1]
        opt.load_state_dict(saved)
    else:
        opt.state.clear()
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    _steps(opt, ps, [7])
    new = optim.AdamW(qs, lr=1e-2)
    _steps(new, qs, [7])
    if how == "partial":
        assert torch.equal(ps[1], qs[1]) and not torch.equal(ps[0], qs[0])
        assert opt.state[ps[1]]["step"] == 1 and opt.state[ps[0]]["step"] == 4
    else:
        _equal(ps, qs)


def test_8_bit_states_start_anew_with_their_scales():
    ps = _params()
    opt = optim.AdamW(ps, state_bits=8)
    _steps(opt, ps, range(2))
    assert all((opt.state[p]["scales"] == 2).all() for p in ps)
    opt.load_state_dict(optim.AdamW(_params(), state_bits=8).state_dict())
    _steps(opt, ps[:1], [3])
    assert (opt.state[ps[0]]["scales"] == 1).all()
