"""The autograd joins of attention and group norm, the flash_attn module under a gradient, and the
example that trains with them.  Numbers of the operators themselves: test_attention_grad_gpu.py,
test_group_norm_grad_gpu.py and test_adamw_gpu.py."""

from __future__ import annotations

import sys

import pytest
import torch
from conftest import REPO

from hi3d_b200 import attention, training, vae
from hi3d_b200.torch_backend import attention as shim

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rand(shape, seed, dtype=torch.float16):
    return torch.randn(shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)).to(dtype)


def test_autograd_hands_back_the_operators_gradients():
    q, k, v = (_rand((2, 4, 70, 64), i).requires_grad_() for i in range(3))
    do = _rand((2, 70, 256), 3)
    out = training.flash_attention(q, k, v, 0.125)
    grads = torch.autograd.grad(out, (q, k, v), do)
    o, lse = attention.flash_attention_lse(q.detach(), k.detach(), v.detach(), 0.125)
    want = attention.flash_attention_backward(do, q.detach(), k.detach(), v.detach(), o, lse, 0.125)
    assert torch.equal(out, o) and all(torch.equal(a, b) for a, b in zip(grads, want))
    x, w, b = _rand((90, 64), 4).requires_grad_(), _rand((64,), 5).requires_grad_(), _rand((64,), 6).requires_grad_()
    y = training.group_norm_act(x, w, b, 8)
    grads = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    y0, mean, rstd = vae.group_norm_act(x.detach(), w, b, 8)
    dx, dw, db = vae.group_norm_act_backward(torch.ones_like(y0), x.detach(), mean, rstd, w, b)
    assert torch.equal(y, y0) and torch.equal(grads[0], dx)
    assert torch.equal(grads[1], dw.half()) and torch.equal(grads[2], db.half())  # in the parameters' type


def test_a_thread_whose_first_cuda_call_is_an_operator():
    """Autograd's threads, and a user's own, begin without a CUDA context."""
    import threading

    q, do = _rand((1, 2, 40, 64), 20), _rand((1, 40, 128), 21)
    out, lse = attention.flash_attention_lse(q, q, q, 0.125)
    want = attention.flash_attention_backward(do, q, q, q, out, lse, 0.125)
    got = []
    t = threading.Thread(target=lambda: got.extend(attention.flash_attention_backward(do, q, q, q, out, lse, 0.125)))
    t.start()
    t.join()
    assert len(got) == 3 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_only_wanted_gradients_and_no_second_order():
    q, k, v = (_rand((1, 2, 20, 64), i) for i in range(3))
    k.requires_grad_()
    out = training.flash_attention(q, k, v, 0.125)
    out.float().sum().backward()  # an expanded gradient
    assert k.grad is not None and q.grad is None and v.grad is None
    q.requires_grad_()
    (g,) = torch.autograd.grad(training.flash_attention(q, k, v, 0.125).float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


@pytest.mark.parametrize("cross", [False, True])
def test_flash_attn_module_under_a_gradient(cross):
    """The module that upstream code calls: the same output with and without a gradient, fused
    gradients equal to the parts'."""
    cu = torch.tensor([0, 40, 130], dtype=torch.int32, device=DEV)
    cu_k = torch.tensor([0, 17, 60], dtype=torch.int32, device=DEV)
    if cross:
        q, kv = _rand((130, 4, 64), 7).requires_grad_(), _rand((60, 2, 4, 64), 8).requires_grad_()
        call = lambda: shim.flash_attn_varlen_kvpacked_func(q, kv, cu, cu_k, 90, 43)  # noqa: E731
        leaves, parts = (q, kv), (q, *kv.unbind(1))
    else:
        qkv = _rand((130, 3, 4, 64), 9).requires_grad_()
        call = lambda: shim.flash_attn_varlen_qkvpacked_func(qkv, cu, 90)  # noqa: E731
        leaves, parts, cu_k = (qkv,), qkv.unbind(1), cu
    out = call()
    with torch.no_grad():
        plain = call()
    assert out.requires_grad and not plain.requires_grad and torch.equal(out, plain)
    do = _rand(out.shape, 10)
    grads = torch.autograd.grad(out, leaves, do)
    other = training.flash_attn_varlen(*parts, cu, cu_k, 90, 0.125)
    want = torch.autograd.grad(other, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    with pytest.raises(NotImplementedError):
        shim.flash_attn_varlen_qkvpacked_func(_rand((4, 3, 1, 64), 11).requires_grad_(), cu[:1], 4, causal=True)


def test_refusals():
    x = _rand((9, 2, 4, 64), 12)
    cu = torch.tensor([0, 9], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        training.flash_attn_varlen_qkvpacked(x, cu, 9, 0.1)
    with pytest.raises(ValueError):
        training.flash_attn_varlen_kvpacked(x[:, 0], x[:, :1], cu, cu, 9, 0.1)


@pytest.mark.parametrize("bits", [32, 8])
def test_example_trains(bits):
    """The loss of fitting a fixed block falls by more than half in 30 steps, to within 20% of what
    the same steps reach with torch's own norm, attention and AdamW (fp32): bf16 and 8-bit states
    may change the path, not the descent."""
    sys.path.insert(0, str(REPO / "examples"))
    import finetune_block as ex

    losses = ex.train(30, state_bits=bits)
    assert losses[-1] < 0.5 * losses[0]

    def norm(x, w, b, groups, offsets=None):
        cuts = (offsets[1:] - offsets[:-1]).tolist()
        return torch.cat([torch.nn.functional.silu(torch.nn.functional.group_norm(s.t()[None], groups, w, b, 1e-6))[0].t()
                          for s in x.split(cuts)])

    def attend(qkv, offsets, longest, scale):
        cuts = (offsets[1:] - offsets[:-1]).tolist()
        rows = []
        for s in qkv.split(cuts):
            q, k, v = s.permute(1, 2, 0, 3)
            rows.append((torch.softmax(q @ k.mT * scale, -1) @ v).transpose(0, 1))
        return torch.cat(rows)

    class Plain:
        group_norm_act = staticmethod(norm)
        flash_attn_varlen_qkvpacked = staticmethod(attend)

    class Torch:
        @staticmethod
        def AdamW(params, state_bits, **kw):
            return torch.optim.AdamW(params, **kw)

    saved = ex.training, ex.optim
    try:
        ex.training, ex.optim = Plain, Torch
        plain = ex.train(30, dtype=torch.float32)
    finally:
        ex.training, ex.optim = saved
    assert losses[-1] < 1.2 * plain[-1]


def test_a_gradient_through_the_convolution_raises():
    """The convolution has no backward pass: a training loop learns of it instead of losing the
    convolution's part of every gradient in silence."""
    from hi3d_b200.torch_backend import sparse_conv

    idx = torch.tensor([[0, x, y, z] for x in range(3) for y in range(3) for z in range(2)], dtype=torch.int32, device=DEV)
    conv = sparse_conv.SubMConv3d(16, 16, 3, indice_key="a").to(DEV, torch.float16)
    x = _rand((idx.shape[0], 16), 30).requires_grad_()
    run = lambda f: conv(sparse_conv.SparseConvTensor(f, idx, [8, 8, 8], 1)).features  # noqa: E731
    out = run(x)
    with torch.no_grad():
        assert torch.equal(run(x), out) and not run(x).requires_grad
    with pytest.raises(NotImplementedError, match="gradient"):
        (x + out).sum().backward()  # a residual block
    with pytest.warns(UserWarning, match="will not be trained"):
        assert not run(x.detach()).requires_grad  # as it was
    conv.requires_grad_(False)
    assert not run(x.detach()).requires_grad
    with pytest.raises(NotImplementedError, match="gradient"):
        run(x).sum().backward()


@pytest.mark.parametrize("grad", [True, False])
def test_flash_attn_module_takes_a_negative_scale(grad):
    """Scores of the other sign, with and without a gradient, on lengths that end inside a block."""
    cu, cu_k = (torch.tensor(c, dtype=torch.int32, device=DEV) for c in ([0, 40, 130], [0, 17, 60]))
    q, kv = _rand((130, 4, 64), 31), _rand((60, 2, 4, 64), 32)
    qkv, do = _rand((130, 3, 4, 64), 33), _rand((130, 4, 64), 34)

    def plain(q, k, v, cut, cut_k):
        rows = []
        for a, b, c, d in zip(cut, cut[1:], cut_k, cut_k[1:]):
            s, e, f = (t.transpose(0, 1) for t in (q[a:b], k[c:d], v[c:d]))
            rows.append((torch.softmax(s @ e.mT * -0.2, -1) @ f).transpose(0, 1))
        return torch.cat(rows)

    for call, leaves, ref in (
            (lambda q, kv: shim.flash_attn_varlen_kvpacked_func(q, kv, cu, cu_k, 90, 43, softmax_scale=-0.2), (q, kv),
             lambda q, kv: plain(q, *kv.unbind(1), [0, 40, 130], [0, 17, 60])),
            (lambda x: shim.flash_attn_varlen_qkvpacked_func(x, cu, 90, softmax_scale=-0.2), (qkv,),
             lambda x: plain(*x.unbind(1), [0, 40, 130], [0, 40, 130]))):
        mine = [t.clone().requires_grad_(grad) for t in leaves]
        theirs = [t.double().requires_grad_() for t in leaves]
        out, want = call(*mine), ref(*theirs)
        # one rounding each of the output and of P, 2^-11 at most, checked as 1.5 of them in the 2-norm
        assert (out.double() - want).norm() <= 1.5 * 2.0 ** -11 * want.norm()
        assert out.requires_grad == grad
        if grad:
            for g, e in zip(torch.autograd.grad(out, mine, do), torch.autograd.grad(want, theirs, do.double())):
                assert (g.double() - e).norm() <= 1.5 * 2.0 ** -11 * e.norm()
