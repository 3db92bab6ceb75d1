"""The optimiser's book-keeping on the CPU: which state a parameter steps on.  The step itself is a plain
AdamW here (on the GPU: test_adamw_gpu.py); the comparisons are bit for bit."""

from __future__ import annotations

import copy
import pickle

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


def test_a_parameter_whose_type_changes_keeps_its_moments():
    """bfloat16 -> float32 -> float16 after steps: the moments and the step count move with the parameter,
    a master is taken from the weights where there was none."""
    ps = _params()
    opt = optim.AdamW(ps, lr=1e-2)
    _steps(opt, ps, range(2))
    for i, dtype in enumerate((torch.bfloat16, torch.float16, torch.float32, torch.bfloat16)):
        before = [{k: v.clone() if torch.is_tensor(v) else v for k, v in opt.state[p].items()} for p in ps]
        for p in ps[:2]:  # the third stays as it was
            p.data = p.data.to(dtype)
        weights = [p.detach().float().clone() for p in ps]
        qs = [torch.nn.Parameter(w.clone()) for w in weights]
        for q, b in zip(qs, before):  # what a float32 optimiser would do on the same moments
            if "master" in b and dtype != torch.float32:
                q.data = b["master"].clone()
        ref = optim.AdamW(qs, lr=1e-2)
        _steps(ref, qs, [50])  # to make its states
        for q, b, w in zip(qs, before, weights):
            q.data = b["master"].clone() if "master" in b and dtype != torch.float32 else w.clone()
            ref.state[q]["exp_avg"].copy_(b["exp_avg"])
            ref.state[q]["exp_avg_sq"].copy_(b["exp_avg_sq"])
            ref.state[q]["step"] = b["step"]
        g = torch.Generator().manual_seed(i)
        for p, q in zip(ps, qs):
            p.grad = torch.randn(p.shape, generator=g).to(p.dtype)
            q.grad = p.grad.float()
        opt.step()
        ref.step()
        for p, q in zip(ps, qs):
            assert torch.equal(p.detach(), q.detach().to(p.dtype)) and opt.state[p]["step"] == ref.state[q]["step"]
            assert ("master" in opt.state[p]) == (p.dtype != torch.float32)


def test_parameters_of_one_group_that_change_one_after_the_other():
    ps = _params()
    opt = optim.AdamW(ps, lr=1e-2)
    _steps(opt, ps, [0])
    for i, p in enumerate(ps):
        p.data = p.data.bfloat16()
        _steps(opt, ps, [i + 1])
        assert torch.equal(p.detach(), opt.state[p]["master"].bfloat16())
    assert [opt.state[p]["step"] for p in ps] == [4, 4, 4]
    assert all((p.detach().abs() > 1e-3).any() for p in ps)


def test_a_parameter_of_another_shape_is_refused():
    ps = _params()
    opt = optim.AdamW(ps)
    _steps(opt, ps, [0])
    ps[0].data = torch.ones(400)
    ps[0].grad = torch.ones(400)
    with pytest.raises(ValueError, match="shape"):
        opt.step()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_a_copied_optimiser_goes_on_by_itself(dtype, how):
    ps = _params(dtype)
    opt = optim.AdamW(ps, lr=1e-2)
    _steps(opt, ps, range(3))
    other = copy.deepcopy(opt) if how == "deepcopy" else pickle.loads(pickle.dumps(opt))
    qs = other.param_groups[0]["params"]
    assert other.state_bits == 32 and all(p is not q for p, q in zip(ps, qs))
    _steps(opt, ps, [5, 6])
    _steps(other, qs, [5, 6])
    _equal(ps, qs)
    _steps(opt, ps, [8])
    assert not torch.equal(ps[0], qs[0]) and opt.state[ps[0]]["step"] == other.state[qs[0]]["step"] + 1


def test_a_parameter_that_grew_before_its_first_step_leaves_its_neighbours_alone():
    ps = _params()
    opt = optim.AdamW(ps, lr=1e-2)
    _steps(opt, ps[1:], [0])
    ps[0].data = torch.ones(700)
    held = opt.state[ps[1]]["exp_avg"].clone()
    ps[1].grad = ps[2].grad = None
    _steps(opt, ps[:1], [1])
    assert torch.equal(opt.state[ps[1]]["exp_avg"], held) and opt.state[ps[0]]["exp_avg"].shape == (700,)


def test_a_load_that_is_refused_changes_nothing():
    ps, qs = _params(), _params()
    a, b = optim.AdamW(ps, lr=1e-2), optim.AdamW(qs, lr=1e-2)
    _steps(a, ps, range(2))
    _steps(b, qs, range(2))
    bad = optim.AdamW(_params(seed=3), lr=0.5)
    _steps(bad, bad.param_groups[0]["params"], [1])
    bad = bad.state_dict()
    bad["state"][2]["exp_avg"] = torch.zeros(3)
    with pytest.raises(ValueError):
        a.load_state_dict(bad)
    _steps(a, ps, [4])
    _steps(b, qs, [4])
    _equal(ps, qs)
