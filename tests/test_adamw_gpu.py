"""The AdamW step against float64 and against torch's own optimiser.

Tolerances.  One step in fp32: the moments are two products and a sum (3 * 2^-24 of their terms),
the update a root, a sum, a quotient and a product of the moments (8 * 2^-24 more, relative), the
weight two products and a sum: 4 * 2^-24 |p| + 16 * 2^-24 |update|.  A 16-bit weight adds its own
rounding.  8-bit states: e4m3 rounds to 2^-4 relative, or 2^-10 of the block's scale below its
normal numbers; the weights of that step do not feel it.
"""

from __future__ import annotations

import pytest
import torch

from hi3d_b200 import _lib, optim

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -24
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [(1,), (255,), (256,), (257,), (3, 1000), (8192,), (70001,), (0,), (127, 129)]


def _rand(shape, seed, dtype=torch.float32):
    return torch.randn(shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)).to(dtype)


def exact(p, g, m, v, step, lr, betas, eps, weight_decay):
    b1, b2 = betas
    p, g, m, v = p.double(), g.double(), m.double(), v.double()
    m0 = m
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    up = lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + eps)
    # what the moment's own rounding (3 * 2^-24 of its terms, which may cancel) moves the weight by
    moved = 3 * E * (b1 * m0.abs() + (1 - b1) * g.abs()) * lr / (1 - b1 ** step) / ((v / (1 - b2 ** step)).sqrt() + eps)
    return p * (1 - lr * weight_decay) - up, m, v, up.abs() + moved / (16 * E)


class Flat:
    """Tensors and flat states made from a seed; values past a tensor's end stay 0."""

    def __init__(self, sizes, dtype, bits, seed=0):
        self.params = [_rand(s, seed + i, dtype) for i, s in enumerate(sizes)]
        self.grads = [_rand(s, seed + 100 + i, dtype) for i, s in enumerate(sizes)]
        self.offsets, self.total = optim.state_layout([p.numel() for p in self.params])
        self.m, self.v = torch.zeros(self.total, device=DEV), torch.zeros(self.total, device=DEV)
        self.master = None if dtype == torch.float32 else torch.zeros(self.total, device=DEV)
        for i, (p, at) in enumerate(zip(self.params, self.offsets)):
            n = p.numel()
            self.m[at:at + n] = _rand((n,), seed + 200 + i) * 0.1
            self.v[at:at + n] = _rand((n,), seed + 300 + i).square() * 0.1
            if self.master is not None:
                self.master[at:at + n] = p.float().view(-1) + _rand((n,), seed + 400 + i) * 1e-4
        self.scales = None
        if bits == 8:
            blocks = lambda t: t.view(-1, optim.BLOCK)  # noqa: E731
            u = self.v.sqrt()
            self.scales = torch.stack([blocks(self.m).abs().amax(1), blocks(u).amax(1)]) / 448
            div = self.scales.clamp_min(1e-30)
            self.m = (blocks(self.m) / div[0, :, None]).to(torch.float8_e4m3fn).view(-1)
            self.v = (blocks(u) / div[1, :, None]).to(torch.float8_e4m3fn).view(-1)

    def values(self):
        """(weights, m, v) of each tensor in float64, from what is held."""
        m, v = self.m.double(), self.v.double()
        if self.scales is not None:
            wide = lambda i: self.scales[i].double().repeat_interleave(optim.BLOCK)  # noqa: E731
            m, v = m * wide(0), (v * wide(1)).square()
        for p, at in zip(self.params, self.offsets):
            n = p.numel()
            w = p if self.master is None else self.master[at:at + n].view(p.shape)
            yield w.double().clone(), m[at:at + n].view(p.shape), v[at:at + n].view(p.shape)

    def step(self, number, **kw):
        optim.adamw_step(self.params, self.grads, self.m, self.v, step=number, master=self.master,
                         scales=self.scales, **(HYPER | kw))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("step", [1, 2, 1000])
def test_one_step_matches_float64(dtype, bits, step):
    f = Flat(SIZES, dtype, bits, seed=step)
    before = [tuple(t.clone() for t in x) for x in f.values()]
    grads = [g.clone() for g in f.grads]
    f.step(step)
    held = list(f.values())
    for i, ((w0, m0, v0), (w, m, v), g) in enumerate(zip(before, held, grads)):
        ew, em, ev, up = exact(w0, g, m0, v0, step, **HYPER)
        assert ((w - ew).abs() <= 4 * E * w0.abs() + 16 * E * up.abs() + 1e-12).all(), i
        terms_m, terms_v = 0.9 * m0.abs() + 0.1 * g.double().abs(), ev
        if bits == 32:
            assert ((m - em).abs() <= 3 * E * terms_m + 1e-30).all() and ((v - ev).abs() <= 4 * E * terms_v + 1e-30).all()
        else:
            at, n = f.offsets[i], w0.numel()
            sm, su = (f.scales[k].double().repeat_interleave(optim.BLOCK)[at:at + n].view(w0.shape) for k in (0, 1))
            assert ((m - em).abs() <= 2.0 ** -4 * em.abs() + 2.0 ** -10 * sm + 1e-6 * terms_m).all()
            u, eu = v.sqrt(), ev.sqrt()
            # a root that is not 0 is held as at least the smallest code
            assert ((u - eu).abs() <= 2.0 ** -4 * eu + 2.0 ** -9 * su + 1e-6 * eu).all() and (u[eu > 0] > 0).all()
        if f.master is not None:
            assert torch.equal(f.params[i].float().view(-1), w.float().to(dtype).float().view(-1))
        assert torch.equal(f.grads[i], grads[i])
    # what lies between the tensors stays 0
    pad = torch.ones(f.total, dtype=torch.bool, device=DEV)
    for p, at in zip(f.params, f.offsets):
        pad[at:at + p.numel()] = False
    for t in (f.m, f.v) + (() if f.master is None else (f.master,)):
        assert not t.float()[pad].any()


def test_hundreds_of_tensors_in_one_call():
    """More tensors than one launch's table holds, the same result as one call each."""
    sizes = [((i * 37) % 700 + 1,) for i in range(1700)]
    a, b = Flat(sizes, torch.bfloat16, 8, seed=7), Flat(sizes, torch.bfloat16, 8, seed=7)
    a.step(3)
    for i in range(len(sizes)):
        optim.adamw_step([b.params[i]], [b.grads[i]], b.m, b.v, step=3, master=b.master, scales=b.scales,
                         offsets=[b.offsets[i]], **HYPER)
    assert all(torch.equal(x, y) for x, y in zip(a.params, b.params))
    assert torch.equal(a.master, b.master) and torch.equal(a.scales, b.scales)
    assert torch.equal(a.m.view(torch.uint8), b.m.view(torch.uint8))
    assert torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.bfloat16, 8)])
def test_unaligned_weights_and_gradients(dtype, bits):
    """Views one element into their storage take the scalar path: the same bits."""
    a, b = Flat([(1000,), (513,)], dtype, bits, seed=9), Flat([(1000,), (513,)], dtype, bits, seed=9)
    for i in range(2):
        for name in ("params", "grads"):
            t = getattr(b, name)[i]
            odd = torch.empty(t.numel() + 1, dtype=dtype, device=DEV)[1:]
            odd.copy_(t)
            getattr(b, name)[i] = odd
    a.step(5)
    b.step(5)
    assert all(torch.equal(x, y) for x, y in zip(a.params, b.params))
    assert torch.equal(a.m.view(torch.uint8), b.m.view(torch.uint8))


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_tiny_and_huge_gradients(bits):
    f = Flat([(1024,)], torch.float32, bits, seed=11)
    f.m.zero_()
    f.v.zero_()
    if f.scales is not None:
        f.scales.zero_()
    w = f.params[0].clone()
    g = f.grads[0]
    g[:256] = 0
    g[256:512] = 1e-36
    g[512:768] *= 1e18
    f.step(1)
    assert all(torch.isfinite(t.float()).all() for t in (f.params[0], f.m, f.v))
    assert torch.equal(f.params[0][:256], w[:256] * torch.tensor(1 - HYPER["lr"] * HYPER["weight_decay"], device=DEV))
    ew = exact(w, g, torch.zeros_like(w), torch.zeros_like(w), 1, **HYPER)[0]
    assert torch.allclose(f.params[0][512:].double(), ew[512:], rtol=1e-6, atol=1e-8)
    f.step(2)
    assert torch.isfinite(f.params[0]).all()


def test_8_bit_codes_are_those_of_correctly_rounded_operations():
    """The states' operations one by one in fp32, each rounded to nearest: every code and scale equal.

    No tolerance: where a root off by one in its last place crosses the middle of two codes, its
    code differs, about once in 3 million values, so ten times here.
    """
    flat = Flat([(1 << 25,)], torch.float32, 8, seed=31)
    f32 = lambda x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    b1, b2 = HYPER["betas"]
    blocks = lambda t: t.view(-1, optim.BLOCK)  # noqa: E731
    scales, g = flat.scales.cpu(), flat.grads[0].cpu()
    m = (blocks(flat.m.cpu().float()) * scales[0][:, None]).view(-1)
    v = (blocks(flat.v.cpu().float()) * scales[1][:, None]).square().view(-1)
    m = m * f32(b1) + g * f32(1 - b1)
    v = v * f32(b2) + (g * g) * f32(1 - b2)
    u = v.double().sqrt().float()  # float32 roots of the CPU may be off by one
    scales = torch.stack([blocks(m).abs().amax(1), blocks(u).amax(1)]) * f32(1 / 448)
    inv = scales.reciprocal()
    c = torch.where(blocks(u) > 0, (blocks(u) * inv[1][:, None]).clamp_min(2.0 ** -9), 0.0)
    flat.step(3)
    assert torch.equal(flat.scales.cpu(), scales)
    code = lambda t: t.to(torch.float8_e4m3fn).view(torch.uint8).view(-1)  # noqa: E731
    assert torch.equal(flat.m.cpu().view(torch.uint8), code(blocks(m) * inv[0][:, None]))
    assert torch.equal(flat.v.cpu().view(torch.uint8), code(c))


def test_a_nan_gradient_spoils_its_own_value_only():
    for bits in (32, 8):
        a, b = Flat([(600,)], torch.float32, bits, seed=12), Flat([(600,)], torch.float32, bits, seed=12)
        b.grads[0][7] = float("nan")
        a.step(2)
        b.step(2)
        keep = torch.arange(600, device=DEV) != 7
        assert torch.isnan(b.params[0][7]) and torch.equal(a.params[0][keep], b.params[0][keep])


def test_grad_scale_multiplies_the_gradients():
    a, b = Flat([(5000,)], torch.float32, 32, seed=13), Flat([(5000,)], torch.float32, 32, seed=13)
    b.grads[0] *= 0.25
    a.step(4, grad_scale=torch.tensor([0.25], device=DEV))
    b.step(4)
    assert torch.equal(a.params[0], b.params[0]) and torch.equal(a.v, b.v)


def _model(dtype, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(37, 65), torch.nn.Linear(65, 20, bias=False)).to(DEV, dtype)


def _set_grads(model, seed):
    for i, p in enumerate(model.parameters()):
        p.grad = _rand(p.shape, seed * 10 + i, p.dtype)


def test_optimiser_follows_torch():
    """Five steps of two groups beside torch.optim.AdamW: each step may differ by the roundings above."""
    ours, theirs = _model(torch.float32), _model(torch.float32)
    groups = lambda m: [{"params": m[0].parameters(), "lr": 1e-2}, {"params": m[1].parameters(), "weight_decay": 0.0}]  # noqa: E731
    a, b = optim.AdamW(groups(ours), lr=2e-3), torch.optim.AdamW(groups(theirs), lr=2e-3)
    for i in range(5):
        _set_grads(ours, i)
        _set_grads(theirs, i)
        if i == 2:  # a parameter without a gradient keeps its step count
            ours[0].bias.grad = theirs[0].bias.grad = None
        a.step()
        b.step()
    assert a.state[ours[0].bias]["step"] == 4 and a.state[ours[0].weight]["step"] == 5
    for p, q in zip(ours.parameters(), theirs.parameters()):
        assert ((p - q).abs() <= 5 * (4 * E * q.abs() + 32 * E * 1e-2)).all()


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.bfloat16, 32), (torch.float16, 8)])
def test_state_dict_continues_bit_for_bit(dtype, bits, tmp_path):
    one, two = _model(dtype), _model(dtype)
    a = optim.AdamW(one.parameters(), lr=1e-2, state_bits=bits)
    for i in range(3):
        _set_grads(one, i)
        a.step()
    torch.save({"model": one.state_dict(), "opt": a.state_dict()}, tmp_path / "s.pt")
    saved = torch.load(tmp_path / "s.pt", weights_only=True)
    two.load_state_dict(saved["model"])
    b = optim.AdamW(two.parameters(), lr=0.5, state_bits=bits)
    b.load_state_dict(saved["opt"])
    assert b.param_groups[0]["lr"] == 1e-2
    for m, o in ((one, a), (two, b)):
        _set_grads(m, 9)
        o.step()
    assert all(torch.equal(p, q) for p, q in zip(one.parameters(), two.parameters()))


def test_small_updates_reach_16_bit_weights_through_the_master():
    """A step of 1e-5 is below half a bf16 step of a weight of 1: 400 of them move it all the same."""
    p = torch.nn.Parameter(torch.ones(300, device=DEV, dtype=torch.bfloat16))
    opt = optim.AdamW([p], lr=1e-5, weight_decay=0.0)
    for _ in range(400):
        p.grad = torch.ones_like(p)
        opt.step()
    assert torch.allclose(opt.state[p]["master"], torch.tensor(1 - 4e-3, device=DEV), atol=1e-5)
    assert (p == torch.tensor(1 - 4e-3).bfloat16().item()).all()


def test_another_stream():
    a, b = Flat([(9000,)], torch.bfloat16, 8, seed=14), Flat([(9000,)], torch.bfloat16, 8, seed=14)
    a.step(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.step(2)
    side.synchronize()
    assert torch.equal(a.params[0], b.params[0]) and torch.equal(a.scales, b.scales)


def test_states_past_32_bit_byte_offsets():
    """A tensor whose fp32 states lie past 2^32 bytes of the flat buffers."""
    at = (1 << 30) + 256
    total = at + 512
    m, v = torch.zeros(total, device=DEV), torch.zeros(total, device=DEV)
    p, g = _rand((500,), 15), _rand((500,), 16)
    w = p.clone()
    optim.adamw_step([p], [g], m, v, step=1, offsets=[at], **HYPER)
    ew, em, ev, up = exact(w, g, torch.zeros_like(w), torch.zeros_like(w), 1, **HYPER)
    assert ((p.double() - ew).abs() <= 4 * E * w.abs() + 16 * E * up.abs() + 1e-12).all()
    assert torch.allclose(m[at:at + 500].double(), em, rtol=1e-6) and not m[at + 500:].any()


def test_refusals():
    f = Flat([(300,)], torch.float32, 32)
    call = lambda **kw: optim.adamw_step(**(dict(params=f.params, grads=f.grads, exp_avg=f.m, exp_avg_sq=f.v, step=1,  # noqa: E731
                                                 **HYPER) | kw))
    for kw in (dict(grads=[]), dict(grads=[f.grads[0].half()]), dict(grads=[f.grads[0][:5]]), dict(step=0),
               dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(exp_avg=f.m[:256]), dict(exp_avg=f.m.half()),
               dict(master=f.m.clone()), dict(scales=torch.ones(2, 2, device=DEV)), dict(offsets=[128]),
               dict(offsets=[1024]), dict(offsets=[0, 0]), dict(params=[f.params[0].cpu()]),
               dict(params=[f.params[0].double()], grads=[f.grads[0].double()]),
               dict(params=[torch.ones(600, device=DEV)[::2]]), dict(grad_scale=torch.ones(1)),
               dict(params=[f.params[0].bfloat16()], grads=[f.grads[0].bfloat16()])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ValueError):
        optim.AdamW([torch.ones(3, device=DEV, dtype=torch.float64, requires_grad=True)])
    with pytest.raises(ValueError):
        optim.AdamW([torch.ones(3, device=DEV, requires_grad=True)], state_bits=16)
    with pytest.raises(ValueError):
        optim.AdamW([torch.ones(3, device=DEV, requires_grad=True)], lr=-1)
    w = torch.ones(3, requires_grad=True)
    w.grad = torch.ones(3)
    with pytest.raises(ValueError):
        optim.AdamW([w]).step()  # not a CUDA tensor
    a = optim.AdamW([torch.ones(300, device=DEV, requires_grad=True)])
    with pytest.raises(ValueError):
        a.load_state_dict(optim.AdamW([torch.ones(3, device=DEV)] * 1, state_bits=8).state_dict() | {"param_groups": []})
    assert _lib.device_status()["code"] == 0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-14])
def test_small_eps_and_tiny_gradients(bits, eps):
    """A v below fp32's normal numbers still has a root: the first step moves each weight by about lr,
    as in torch's optimiser.  Expected from the fp32 moments (a subnormal v has few bits), the rest in
    float64: the root, product, sum, quotient and product of the update, 16 * 2^-24 of it."""
    f = Flat([(4096,)], torch.float32, bits, seed=41)
    for t in (f.m, f.v) + (() if f.scales is None else (f.scales,)):
        t.zero_()
    g = torch.logspace(-20.5, -15, 4096, device=DEV) * torch.where(torch.arange(4096, device=DEV) % 2 == 0, 1, -1)
    f.grads[0].copy_(g)
    w = f.params[0].double()
    b1, b2, lr = 0.9, 0.999, HYPER["lr"]
    f.step(1, eps=eps, betas=(b1, b2))
    f32 = lambda x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    c = g.cpu()
    m, v = c * f32(1 - b1), (c * c) * f32(1 - b2)  # the CPU keeps subnormals
    up = (m.double() * (lr / (1 - b1)) / (v.double().sqrt() * (1 - b2) ** -0.5 + eps)).to(DEV)
    want = w * (1 - lr * HYPER["weight_decay"]) - up
    assert torch.isfinite(f.params[0]).all()
    assert ((f.params[0].double() - want).abs() <= 4 * E * w.abs() + 16 * E * up.abs() + 1e-12).all()


def test_a_backward_pass_over_weights_that_a_step_changed_raises():
    p = torch.nn.Parameter(_rand((16, 16), 51))
    x = _rand((4, 16), 52).requires_grad_()
    opt = optim.AdamW([p])
    y = x @ p
    y.sum().backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    f = Flat([(300,)], torch.bfloat16, 8)
    held = [f.params[0], f.m, f.v, f.master, f.scales]
    before = [t._version for t in held]
    f.step(1)
    assert all(t._version > b for t, b in zip(held, before)) and f.grads[0]._version == 0


def test_states_in_another_order():
    """Offsets that fall, with an empty tensor inside another's state: the same step as in order."""
    a, b = Flat([(300,), (0,), (256,), (5,)], torch.float32, 32, seed=61), Flat([(300,), (0,), (256,), (5,)],
                                                                                  torch.float32, 32, seed=61)
    b.m, b.v = (torch.cat([t[768:], t[512:768], t[:512]]) for t in (b.m, b.v))
    a.step(3)
    b.step(3, offsets=[512, 512, 256, 0])
    assert all(torch.equal(p, q) for p, q in zip(a.params, b.params))
    assert torch.equal(torch.cat([b.m[512:], b.m[256:512], b.m[:256]]), a.m)
