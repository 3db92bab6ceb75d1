"""Attention's training pair (forward with log-sum-exp, backward) against float64.

Tolerances.  u = 2^-8 (bf16) or 2^-11 (fp16) is the largest relative error of one rounding; its
root mean square over random values is about 0.45 u.  An output value carries the rounding of the
output itself, of P or dS as an operand (independent errors over the terms of a sum, so the same
relative size) and, through delta, of the saved output: three in all, 0.78 u in quadrature, checked
as 1.5 u in the 2-norm.  What cancels exactly (one key: dS = 0) leaves fp32 rounding, covered by
an absolute part of 1e-5 times the 2-norm of the terms' size.  The log-sum-exp is fp32 throughout:
scores of D products (D 2^-24 relative to sum |q k|), the exponential's 3e-6.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from hi3d_b200 import _lib, attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _rand(shape, dtype, seed, mul=1.0):
    g = torch.Generator(DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * mul).to(dtype)


def exact(q, k, v, do, scale):
    """float64 (out, lse, dq, dk, dv) of q, do [B, H, Nq, D] and k, v [1 or B, Hk, Nk, D], from the
    formulas."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    g = q.shape[1] // k.shape[1]
    kk, vv = (t.repeat_interleave(g, 1) for t in (k, v))
    if k.shape[2] == 0:
        return (torch.zeros_like(q), torch.full(q.shape[:3], -math.inf, device=q.device), torch.zeros_like(q),
                torch.zeros_like(k), torch.zeros_like(v))
    s = q @ kk.mT * scale
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    out = p @ vv
    dp = do @ vv.mT
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale

    def fold(t):
        t = t.unflatten(1, (k.shape[1], g)).sum(2)
        return t.sum(0, keepdim=True) if k.shape[0] == 1 else t

    return out, lse, ds @ kk, fold(ds.mT @ q), fold(p.mT @ do)


def check(name, got, want, dtype, size=1.0):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all(), name
    tol = 1.5 * U[dtype] * want.norm() + 1e-5 * size * math.sqrt(max(1, want.numel()))
    err = (got - want).norm()
    assert err <= tol, f"{name}: {err:.3e} > {tol:.3e} (norm {want.norm():.3e})"


def check_all(got, want, dtype):
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        check(name, a, b, dtype)


def dense(q, k, v, do, scale, layout="bhnd", **kw):
    """(out, lse, dq, dk, dv) through the operators, as [B, H, N, D]."""
    b, h, n, d = q.shape
    qq = q if layout == "bhnd" else q.transpose(1, 2).contiguous()
    out, lse = attention.flash_attention_lse(qq, k, v, scale, layout)
    flat = do.transpose(1, 2).reshape(b, n, h * d)
    dq, dk, dv = attention.flash_attention_backward(flat, qq, k, v, out, lse, scale, layout, **kw)
    if layout == "bnhd":
        dq = dq.transpose(1, 2)
    return out.view(b, n, h, d).transpose(1, 2), lse, dq, dk, dv


def compare(q, k, v, do, scale, layout="bhnd"):
    out, lse, dq, dk, dv = dense(q, k, v, do, scale, layout)
    e = exact(q, k, v, do, scale)
    check_all((out, dq, dk, dv), (e[0], *e[2:]), q.dtype)
    assert torch.allclose(lse.double(), e[1], rtol=1e-5, atol=2e-5)
    assert _lib.device_status()["code"] == 0


SIZES = [(1, 2), (1, 300), (3, 5), (64, 64), (127, 129), (128, 128), (129, 127), (257, 1000), (700, 65), (1000, 1370)]


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,nk", SIZES)
def test_gradients_match_float64(dim, dtype, nq, nk):
    q, do = _rand((2, 3, nq, dim), dtype, 1), _rand((2, 3, nq, dim), dtype, 2)
    k, v = _rand((2, 3, nk, dim), dtype, 3), _rand((2, 3, nk, dim), dtype, 4)
    compare(q, k, v, do, dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads,batch,shared", [(8, 2, 1, False), (6, 1, 2, True), (4, 4, 3, True),
                                                         (4, 2, 2, False)])
def test_grouped_heads_and_shared_keys_sum_their_gradients(dim, heads, kv_heads, batch, shared):
    dtype = torch.bfloat16
    q, do = _rand((batch, heads, 333, dim), dtype, 5), _rand((batch, heads, 333, dim), dtype, 6)
    shape = (1 if shared else batch, kv_heads, 201, dim)
    compare(q, _rand(shape, dtype, 7), _rand(shape, dtype, 8), do, dim ** -0.5, "bnhd")


@pytest.mark.parametrize("nq,nk", [(6000, 77), (3, 9000), (40, 40)])
def test_few_tiles_split_their_streams(nq, nk):
    """A short key set under many queries, and few queries over many keys, run split with fp32
    partials: the same bounds, the same bits on every run."""
    dtype = torch.float16
    q, do = _rand((1, 2, nq, 64), dtype, 9), _rand((1, 2, nq, 64), dtype, 10)
    k, v = _rand((1, 2, nk, 64), dtype, 11), _rand((1, 2, nk, 64), dtype, 12)
    compare(q, k, v, do, 0.125)
    a, b = dense(q, k, v, do, 0.125), dense(q, k, v, do, 0.125)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_one_key_has_no_score_gradient():
    """P = 1 whatever the scores: dq = dk = 0 up to fp32 rounding of dP - delta (64 products of
    unit values: 64 * 2^-24 * 8 * scale), dv the sum of the gradients."""
    q, do = _rand((1, 2, 70, 64), torch.float16, 13), _rand((1, 2, 70, 64), torch.float16, 14)
    k, v = _rand((1, 2, 1, 64), torch.float16, 15), _rand((1, 2, 1, 64), torch.float16, 16)
    out, lse, dq, dk, dv = dense(q, k, v, do, 0.125)
    assert dq.abs().max() <= 2e-5 and dk.abs().max() <= 70 * 2e-5
    check("dv", dv, do.double().sum(2, keepdim=True), torch.float16)
    assert torch.equal(out, v.expand_as(out))


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (96, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("nk", [2, 3, 7, 16, 17])
def test_few_keys_keep_their_bits(dim, dtype, nk):
    """Over a few keys delta nearly cancels dP, so that the saved output's rounding would be most of
    dS's error.  Without it a score gradient carries two roundings, of dS and its own: 0.64 u in
    quadrature, checked at 0.8 u.  From 17 keys on the output's is small beside them.  A dense set,
    and a sequence beside others of one and no key."""
    q, do = _rand((2, 3, 700, dim), dtype, 41), _rand((2, 3, 700, dim), dtype, 42)
    k, v = _rand((2, 3, nk, dim), dtype, 43), _rand((2, 3, nk, dim), dtype, 44)

    def close(name, got, want):
        err, tol = (got.double() - want).norm(), 0.8 * U[dtype] * want.norm()
        assert err <= tol, f"{name}: {err:.3e} > {tol:.3e}"

    out, lse, dq, dk, dv = dense(q, k, v, do, dim ** -0.5)
    e = exact(q, k, v, do, dim ** -0.5)
    close("dq", dq, e[2])
    close("dk", dk, e[3])
    one = lambda t: t[0].transpose(0, 1).contiguous()  # noqa: E731
    cu_q, cu_k = [0, 5, 5, 700], [0, 1, 1, nk + 1]
    kk, vv = (torch.cat([one(t)[:1], one(t)]) for t in (k, v))
    got = packed(one(q), kk, vv, one(do), cu_q, cu_k, dim ** -0.5)
    e = exact(q[:1, :, 5:], k[:1], v[:1], do[:1, :, 5:], dim ** -0.5)
    close("packed dq", got[2][5:], e[2][0].transpose(0, 1))
    close("packed dk", got[3][1:], e[3][0].transpose(0, 1))


@pytest.mark.parametrize("mul", [1e-4, 1e-2, 300.0])
def test_fp16_gradients_of_any_size_keep_their_bits(mul):
    """dS = P (dP - delta) is far below fp16's normal range for small gradients over many keys and
    above it for large ones; its power-of-two scale follows max |dO| max |V|.  The bound is
    relative to each gradient, for values that fp16 itself holds as normal numbers: v and k
    are large where the output gradient is small."""
    n = 4096
    q, do = _rand((1, 1, n, 64), torch.float16, 17), _rand((1, 1, n, 64), torch.float16, 18, mul)
    up = 1.0 if mul > 1 else 16.0
    k, v = _rand((1, 1, n, 64), torch.float16, 19), _rand((1, 1, n, 64), torch.float16, 20, up)
    q, k = (q, k) if mul > 1 else (q * 8, k)
    out, lse, dq, dk, dv = dense(q, k, v, do, 0.125)
    e = exact(q, k, v, do, 0.125)
    for name, a, b in (("dq", dq, e[2]), ("dk", dk, e[3]), ("dv", dv, e[4])):
        tiny = 2.0 ** -25 * math.sqrt(b.numel())  # half of fp16's smallest step, where a value is subnormal
        err = (a.double() - b).norm()
        assert err <= 1.5 * U[torch.float16] * b.norm() + tiny, (name, float(err), float(b.norm()))


def packed_exact(q, k, v, do, cu_q, cu_k, scale):
    out, dq = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    dk, dv = torch.zeros_like(k, dtype=torch.float64), torch.zeros_like(v, dtype=torch.float64)
    lse = torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    for n in range(len(cu_q) - 1):
        a, b = cu_q[n], cu_q[n + 1]
        c, d = (0, k.shape[0]) if cu_k is None else (cu_k[n], cu_k[n + 1])
        if a == b or c == d:
            continue
        side = lambda t, lo, hi: t[lo:hi].transpose(0, 1)[None]  # noqa: E731
        r = exact(side(q, a, b), side(k, c, d), side(v, c, d), side(do, a, b), scale)
        back = lambda t: t[0].transpose(0, 1)  # noqa: E731
        out[a:b], lse[:, a:b], dq[a:b] = back(r[0]), r[1][0], back(r[2])
        dk[c:d] += back(r[3])
        dv[c:d] += back(r[4])
    return out, lse, dq, dk, dv


def packed(q, k, v, do, cu_q, cu_k, scale, **kw):
    cq = torch.tensor(cu_q, dtype=torch.int32, device=DEV)
    ck = None if cu_k is None else torch.tensor(cu_k, dtype=torch.int32, device=DEV)
    longest = max(b - a for a, b in zip(cu_q, cu_q[1:]))
    out, lse = attention.flash_attn_varlen_lse(q, k, v, cq, ck, longest, scale)
    return (out, lse, *attention.flash_attn_varlen_backward(do, q, k, v, out, lse, cq, ck, scale, **kw))


RAGGED = [([0, 100, 100, 357, 700, 701], [0, 100, 100, 357, 700, 701]),       # an empty sequence, one row
          ([0, 128, 256, 300], [0, 0, 77, 205]),                              # queries without keys
          ([0, 0, 5, 5, 260], [0, 130, 140, 300, 428]),                       # keys without queries
          ([0, 333], [0, 129]), ([0, 200, 450], None), ([0, 1, 2, 3, 4], [0, 1, 3, 6, 10])]


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (96, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("cu_q,cu_k", RAGGED)
def test_packed_sequences_match_float64(dim, dtype, cu_q, cu_k):
    tk = 391 if cu_k is None else cu_k[-1]
    q, do = _rand((cu_q[-1], 4, dim), dtype, 21), _rand((cu_q[-1], 4, dim), dtype, 22)
    kv = _rand((tk, 2, 2, dim), dtype, 23)
    k, v = kv.unbind(1)  # views of a fused projection
    got = packed(q, k, v, do, cu_q, cu_k, dim ** -0.5)
    want = packed_exact(q, k, v, do, cu_q, cu_k, dim ** -0.5)
    check_all((got[0], *got[2:]), (want[0], *want[2:]), dtype)
    empty = torch.isinf(want[1])
    assert torch.equal(torch.isinf(got[1]) & (got[1] < 0), empty)
    assert torch.allclose(got[1][~empty].double(), want[1][~empty], rtol=1e-5, atol=2e-5)
    gone = empty.all(0)
    assert not got[0][gone].any() and not got[2][gone].any()
    assert _lib.device_status()["code"] == 0


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (96, torch.bfloat16)])
def test_a_neighbour_sequence_full_of_nan_or_infinities_does_not_leak(dim, dtype, bad):
    cu = [0, 70, 200, 463]
    qkv, do = _rand((463, 3, 2, dim), dtype, 24), _rand((463, 2, dim), dtype, 25)
    qkv[70:200], do[70:200] = bad, bad
    q, k, v = qkv.unbind(1)
    got = packed(q, k, v, do, cu, cu, dim ** -0.5)
    keep = torch.cat([torch.arange(0, 70), torch.arange(200, 463)]).to(DEV)
    part = [t[keep] for t in (q, k, v, do)]
    want = packed_exact(*part, [0, 70, 333], [0, 70, 333], dim ** -0.5)
    check_all([t[keep] for t in (got[0], *got[2:])], (want[0], *want[2:]), dtype)
    assert torch.isfinite(got[1][:, keep]).all()


def test_sharp_rows_and_scores_of_the_largest_size():
    """Scores up to +-1e4 and a few at -6e7: rows with one probability near 1, where dP - delta is a
    small difference.  Checked value by value against the sum of each term's own rounding: a score of
    size s is off by up to 2^-21 s (fp32 products and sums, log-sum-exp, scaling), so P by that
    relatively; P and dS are rounded (u); delta = dO O carries O's rounding and the P inside O, up to
    2 u sum |dO| P |V|; the result is rounded (u)."""
    u, scale = U[torch.float16], 1.0
    q, do = _rand((1, 2, 130, 64), torch.float16, 26, 20.0), _rand((1, 2, 130, 64), torch.float16, 27)
    k, v = _rand((1, 2, 200, 64), torch.float16, 28, 20.0), _rand((1, 2, 200, 64), torch.float16, 29)
    q[0, 0, 3] = 0
    k[0, 1, :5] = 60000.0
    q[0, 1] = q[0, 1].abs().neg()  # the large keys score lowest in the second head
    out, lse, dq, dk, dv = dense(q, k, v, do, scale)
    e = exact(q, k, v, do, scale)
    qd, kd, vd, dd = (t.double() for t in (q, k, v, do))
    s = qd @ kd.mT * scale
    p = torch.exp(s - e[1][..., None])
    eps = 2.0 ** -21 * torch.maximum(s.abs(), e[1].abs()[..., None]) + 1e-5
    p = p * torch.exp(eps.clamp_max(1.0))  # the largest the kernel's P can be
    diff = dd @ vd.mT
    diff = (diff - (p * diff).sum(-1, keepdim=True)).abs() + 1e-4
    delta = 2 * u * (dd.abs() * (p @ vd.abs())).sum(-1, keepdim=True)
    ds = p * ((2 * u + 2 * eps.clamp_max(1.0)) * diff + delta + (eps * p).sum(-1, keepdim=True) * diff) * scale
    ds = ds + 2.0 ** -24  # a dS below fp16's normal numbers
    for name, got, want, bound in (("dq", dq, e[2], ds @ kd.abs()), ("dk", dk, e[3], ds.mT @ qd.abs()),
                                   ("dv", dv, e[4], ((u + eps) * p).mT @ dd.abs())):
        assert torch.isfinite(got).all(), name
        assert ((got.double() - want).abs() <= bound + 2 * u * want.abs() + 1e-6).all(), name
    assert _lib.device_status()["code"] == 0


def test_strided_inputs_gradients_and_expanded_output_gradient():
    """Heads in the middle of a wider row, gradients written into views of one fused tensor, and
    the expanded gradient that .sum() hands back."""
    big = _rand((2, 150, 3, 8, 64), torch.bfloat16, 30)
    q, k, v = (big[:, :, i, 1:7].transpose(1, 2) for i in range(3))
    out, lse = attention.flash_attention_lse(q, k, v, 0.125)
    ones = torch.ones((), dtype=torch.bfloat16, device=DEV).expand(2, 150, 6 * 64)
    fused = torch.full((2, 150, 3, 8, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    grads = tuple(fused[:, :, i, 1:7].transpose(1, 2) for i in range(3))
    got = attention.flash_attention_backward(ones, q, k, v, out, lse, 0.125, grads=grads)
    assert all(a is b for a, b in zip(got, grads))
    e = exact(q, k, v, torch.ones_like(q), 0.125)
    check_all((out.view(2, 150, 6, 64).transpose(1, 2), *got), (e[0], *e[2:]), torch.bfloat16)
    assert (fused[:, :, :, 0] == 7).all() and (fused[:, :, :, 7] == 7).all()


def test_row_offsets_past_32_bits():
    """Rows 2^22 elements apart: element offsets reach 2^32 (8.6 GB spanned by each tensor)."""
    step, n = 1 << 22, 1030
    store = torch.empty(n * step, dtype=torch.bfloat16, device=DEV)
    view = lambda at: store.as_strided((1, 1, n, 64), (step, 64, step, 1), at)  # noqa: E731
    q, k, v, dq, dk, dv = (view(i * 64) for i in range(6))
    for i, t in enumerate((q, k, v)):
        t.copy_(_rand((1, 1, n, 64), torch.bfloat16, 31 + i))
    do = _rand((1, 1, n, 64), torch.bfloat16, 34)
    out, lse = attention.flash_attention_lse(q, k, v, 0.125)
    attention.flash_attention_backward(do.view(1, n, 64), q, k, v, out, lse, 0.125, grads=(dq, dk, dv))
    e = exact(q, k, v, do, 0.125)
    check_all((out.view(1, 1, n, 64), dq, dk, dv), (e[0], *e[2:]), torch.bfloat16)


def test_gradients_match_differences():
    """Central differences of the float64 attention along a random direction of (q, k, v) against
    <gradient, direction>: 1.5 u of the gradient's norm times the direction's, as above."""
    q, do = _rand((1, 2, 90, 64), torch.bfloat16, 35), _rand((1, 2, 90, 64), torch.bfloat16, 36)
    k, v = _rand((1, 1, 140, 64), torch.bfloat16, 37), _rand((1, 1, 140, 64), torch.bfloat16, 38)
    _, _, *grads = dense(q, k, v, do, 0.125)
    step = [_rand(t.shape, torch.float64, 39 + i) for i, t in enumerate((q, k, v))]
    f = lambda e: (exact(*(t.double() + e * s for t, s in zip((q, k, v), step)), do, 0.125)[0] * do.double()).sum()  # noqa: E731
    diff = (f(1e-4) - f(-1e-4)) / 2e-4
    got = sum((g.double() * s).sum() for g, s in zip(grads, step))
    bound = 1.5 * U[torch.bfloat16] * math.sqrt(sum(float(g.double().norm() ** 2) for g in grads))
    # the errors are independent of the direction: their inner product has the size of one coordinate
    assert abs(got - diff) <= 6 * bound


def test_no_keys_no_queries_no_batch():
    q, k = _rand((2, 3, 5, 64), torch.float16, 40), _rand((2, 3, 0, 64), torch.float16, 41)
    out, lse = attention.flash_attention_lse(q, k, k, 0.125)
    assert not out.any() and (lse == -math.inf).all()
    dq, dk, dv = attention.flash_attention_backward(torch.ones_like(out), q, k, k, out, lse, 0.125)
    assert not dq.any() and dk.shape == k.shape and dv.shape == k.shape
    q, k = _rand((2, 3, 0, 64), torch.float16, 42), _rand((2, 3, 9, 64), torch.float16, 43)
    out, lse = attention.flash_attention_lse(q, k, k, 0.125)
    dq, dk, dv = attention.flash_attention_backward(out, q, k, k, out, lse, 0.125)
    assert dq.shape == q.shape and not dk.any() and not dv.any()
    cu = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = _rand((0, 2, 64), torch.float16, 44)
    out, lse = attention.flash_attn_varlen_lse(q, q, q, cu, cu, 0, 0.125)
    assert out.shape == q.shape and lse.shape == (2, 0)


def test_a_scale_of_zero_attends_evenly():
    q, k, v, do = (_rand((1, 2, 40 + 9 * i, 64), torch.bfloat16, 60 + i) for i in range(4))
    v, do = v[:, :, :49], do[:, :, :40]
    out, lse, dq, dk, dv = dense(q, k, v, do, 0.0)
    assert torch.allclose(lse, torch.tensor(math.log(49.0), device=DEV), rtol=1e-6)
    assert not dq.any() and not dk.any()
    check("dv", dv, (do.double().sum(2, keepdim=True) / 49).expand_as(dv), torch.bfloat16)


def test_saved_tensors_in_other_layouts():
    """out and its gradient as views of wider rows, lse with strides of its own: the same bits."""
    q, k, v, do = (_rand((2, 3, 50, 64), torch.float16, 70 + i) for i in range(4))
    want = dense(q, k, v, do, 0.125)
    out, lse = attention.flash_attention_lse(q, k, v, 0.125)
    wide = torch.zeros((2, 50, 400), dtype=torch.float16, device=DEV)
    wide[..., 8:200], wide[..., 200:392] = out, do.transpose(1, 2).flatten(2)
    apart = torch.empty((50, 2, 3), device=DEV).permute(1, 2, 0).copy_(lse)
    got = attention.flash_attention_backward(wide[..., 200:392], q, k, v, wide[..., 8:200], apart, 0.125)
    assert all(torch.equal(a, b) for a, b in zip(got, want[2:]))
    slow = torch.empty((192, 2, 50), dtype=torch.float16, device=DEV).permute(1, 2, 0).copy_(out)
    got = attention.flash_attention_backward(wide[..., 200:392], q, k, v, slow, lse, 0.125)
    assert all(torch.equal(a, b) for a, b in zip(got, want[2:]))


def test_another_stream_and_odd_alignment():
    q, k, v, do = (_rand((1, 2, 200, 64), torch.float16, 45 + i) for i in range(4))
    want = dense(q, k, v, do, 0.125)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape)  # 2 bytes past an aligned address
    odd.copy_(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dense(odd, k, v, do, 0.125)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    q = _rand((1, 4, 8, 64), torch.float16, 50)
    k3, k64 = _rand((1, 3, 8, 64), torch.float16, 51), _rand((1, 4, 8, 64), torch.bfloat16, 52)
    with pytest.raises(ValueError):
        attention.flash_attention_lse(q, k3, k3, 0.1)          # 3 key heads under 4
    with pytest.raises(ValueError):
        attention.flash_attention_lse(q, k64, k64, 0.1)        # two dtypes
    with pytest.raises(ValueError):
        attention.flash_attention_lse(q.float(), q.float(), q.float(), 0.1)
    for scale in (-0.1, math.nan, math.inf):
        with pytest.raises(ValueError):
            attention.flash_attention_lse(q, q, q, scale)
    with pytest.raises(ValueError):
        attention.flash_attention_lse(q, q, q, 0.1, "hbnd")
    with pytest.raises(ValueError):
        attention.flash_attention_lse(q, q, q, 0.1, "packed")
    with pytest.raises(NotImplementedError):
        attention.flash_attention_lse(q[..., :32], q[..., :32], q[..., :32], 0.1)
    with pytest.raises(ValueError):
        attention.flash_attention_lse(q.cpu(), q, q, 0.1)
    out, lse = attention.flash_attention_lse(q, q, q, 0.1)
    with pytest.raises(ValueError):
        attention.flash_attention_backward(out[:, :4], q, q, q, out, lse, 0.1)
    with pytest.raises(ValueError):
        attention.flash_attention_backward(out, q, q, q, out, lse.half(), 0.1)
    with pytest.raises(ValueError):
        attention.flash_attention_backward(out, q, q, q, out, lse, 0.1, grads=(q[..., :4], None, None))
    t = q[0].transpose(0, 1)
    cu = torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        attention.flash_attn_varlen_lse(t, t, t, cu, cu[:1], 8, 0.1)
    with pytest.raises(ValueError):
        attention.flash_attn_varlen_lse(t, t, t, cu.float(), cu, 8, 0.1)
    with pytest.raises(ValueError):
        attention.flash_attn_varlen_lse(t, t, t, cu, cu, 0, 0.1)


def _poison(nbytes):
    """Leaves NaN bits in the block of memory that the next workspace of this size is given."""
    torch.full((nbytes,), 0xFF, dtype=torch.uint8, device=DEV)


# 2 heads over many queries and few keys split the key stream, 2 queries' tiles over many keys the query
# stream; the last is whole.  Rows before the first, after the last offset belong to no sequence.
UNCOVERED = [([5, 3000, 6000], 6100, [3, 77, 150], 256), ([2, 3, 5], 9, [0, 100, 9000], 9100),
             ([5, 100, 190], 200, [3, 77, 150], 256)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cu_q,tq,cu_k,tk", UNCOVERED)
def test_gradient_rows_of_no_sequence_are_not_written(dtype, cu_q, tq, cu_k, tk):
    q, do = _rand((tq, 2, 64), dtype, 81), _rand((tq, 2, 64), dtype, 82)
    k, v = _rand((tk, 2, 64), dtype, 83), _rand((tk, 2, 64), dtype, 84)
    cq, ck = (torch.tensor(c, dtype=torch.int32, device=DEV) for c in (cu_q, cu_k))
    out, lse = attention.flash_attn_varlen_lse(q, k, v, cq, ck, max(b - a for a, b in zip(cu_q, cu_q[1:])), 0.125)
    grads = tuple(torch.full_like(t, 7.0) for t in (q, k, v))
    p = attention._planned("packed", q, k, v)[0]
    steps = (128, 64, 0) * 2
    _poison(attention._backward_plan(p, q.shape, k.shape, steps, True, len(cu_q) - 1, 0.125, 0)[2])
    dq, dk, dv = attention.flash_attn_varlen_backward(do, q, k, v, out, lse, cq, ck, 0.125, grads=grads)
    for t, cu in ((dq, cu_q), (dk, cu_k), (dv, cu_k)):
        assert (t[:cu[0]] == 7).all() and (t[cu[-1]:] == 7).all()
    rows = lambda t, cu: t[cu[0]:cu[-1]]  # noqa: E731
    zero = lambda cu: [c - cu[0] for c in cu]  # noqa: E731
    want = packed_exact(rows(q, cu_q), rows(k, cu_k), rows(v, cu_k), rows(do, cu_q), zero(cu_q), zero(cu_k), 0.125)
    for name, got, e in (("dq", rows(dq, cu_q), want[2]), ("dk", rows(dk, cu_k), want[3]), ("dv", rows(dv, cu_k), want[4])):
        check(name, got, e, dtype)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("with_lse", [True, False])
def test_output_rows_of_no_sequence_are_not_written(splits, with_lse):
    """The C entry on buffers of the caller's: rows outside the offsets keep what they held, with the
    keys in one pass or split."""
    tq, tk, heads, cu_q, cu_k = 300, 900, 2, [5, 100, 290], [3, 400, 890]
    dtype = torch.bfloat16
    q, k, v = (_rand((n, heads, 64), dtype, 85 + i) for i, n in enumerate((tq, tk, tk)))
    cq, ck = (torch.tensor(c, dtype=torch.int32, device=DEV) for c in (cu_q, cu_k))
    out, lse = torch.full_like(q, 7.0), torch.full((heads, tq), 7.0, device=DEV)
    args = _lib.AttnArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), *(128, 64, 0) * 4, cq.data_ptr(),
                         ck.data_ptr(), tq, tk, 190, 2, heads, 64, _lib.BF16, 0.125)
    nbytes = ctypes.c_int64()
    lib = _lib.load()
    _lib.check(lib.hi3d_flash_attn_split_workspace_size(ctypes.byref(args), splits, ctypes.byref(nbytes)), "size")
    ws = torch.full((max(1, nbytes.value),), 0x40, dtype=torch.uint8, device=DEV)  # floats of about 3
    if with_lse:
        rc = lib.hi3d_flash_attn_fwd_lse(ctypes.byref(args), heads, lse.data_ptr(), splits, ws.data_ptr(), nbytes.value,
                                         _lib.stream(q))
    else:
        rc = lib.hi3d_flash_attn_fwd_split(ctypes.byref(args), splits, ws.data_ptr(), nbytes.value, _lib.stream(q))
    _lib.check(rc, "forward")
    gone = torch.ones(tq, dtype=torch.bool, device=DEV)
    gone[5:290] = False
    assert (out[gone] == 7).all() and (lse[:, gone] == 7).all()
    want = packed_exact(q[5:290], k[3:890], v[3:890], q[5:290], [0, 95, 285], [0, 397, 887], 0.125)
    check("out", out[5:290], want[0], dtype)
    if with_lse:
        assert torch.allclose(lse[:, 5:290].double(), want[1], rtol=1e-5, atol=2e-5)


def _each_by_its_own(got, want):
    """Bounds relative to each gradient's own norm, plus half of fp16's smallest step."""
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        a, b = a.double(), b.double()
        assert torch.isfinite(a).all(), name
        err, tol = (a - b).norm(), 1.5 * U[torch.float16] * b.norm() + 2.0 ** -25 * math.sqrt(b.numel())
        assert err <= tol, f"{name}: {err:.3e} > {tol:.3e} (norm {b.norm():.3e})"


@pytest.mark.parametrize("v_mul,do_mul", [(75.0, 0.01), (6000.0, 0.1), (6000.0, 0.01)])
@pytest.mark.parametrize("kv_heads", [2, 1])
def test_fp16_gradients_of_a_sequence_do_not_depend_on_its_neighbours_sizes(v_mul, do_mul, kv_heads):
    """A sequence of 2048 rows beside one with values and output gradients many times its own, and
    beside rows that no sequence reads: its gradients keep the bits that they have alone."""
    dtype, cu = torch.float16, [0, 2048, 2400]
    q, do = _rand((2464, 2, 64), dtype, 91), _rand((2464, 2, 64), dtype, 92)
    k, v = _rand((2464, kv_heads, 64), dtype, 93), _rand((2464, kv_heads, 64), dtype, 94)
    v[2048:] *= v_mul
    v[2400:] = 60000.0
    do[:2048] *= do_mul
    do[2400:] = 60000.0
    got = packed(q, k, v, do, cu, cu, 0.125)
    own = [t[:2048] for t in (q, k, v, do)]
    want = packed_exact(*own, [0, 2048], [0, 2048], 0.125)
    _each_by_its_own([t[:2048] for t in got[2:]], want[2:])
    alone = packed(*own, [0, 2048], [0, 2048], 0.125)
    _each_by_its_own([t[:2048] for t in got[2:]], alone[2:])


@pytest.mark.parametrize("which", ["head", "batch"])
def test_fp16_gradients_of_a_head_do_not_depend_on_the_others_sizes(which):
    dtype = torch.float16
    q, k, v, do = (_rand((2, 2, 1500, 64), dtype, 95 + i) for i in range(4))
    big = (slice(None), 1) if which == "head" else (1,)
    v[big] *= 6000.0
    do *= 0.01
    do[big] *= 400.0
    out, lse, *got = dense(q, k, v, do, 0.125)
    want = exact(q, k, v, do, 0.125)[2:]
    small = (slice(None), 0) if which == "head" else (0,)
    _each_by_its_own([t[small] for t in got], [t[small] for t in want])


def test_fp16_query_gradients_do_not_depend_on_other_rows_sizes():
    """One row tile whose output gradient is thousands of times the others'."""
    q, k, v, do = (_rand((1, 2, 2000, 64), torch.float16, 99 + i) for i in range(4))
    do *= 1e-3
    do[:, :, 256:384] *= 1e6
    v *= 40.0
    out, lse, dq, *_ = dense(q, k, v, do, 0.125)
    want = exact(q, k, v, do, 0.125)[2]
    rest = torch.ones(2000, dtype=torch.bool, device=DEV)
    rest[256:384] = False
    _each_by_its_own([dq[:, :, rest]], [want[:, :, rest]])


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (64, torch.bfloat16), (128, torch.bfloat16)])
@pytest.mark.parametrize("nq,nk", [(130, 300), (3, 9000), (70, 7)])
@pytest.mark.parametrize("at", [0, 1, 2])
def test_a_nan_reaches_all_that_depends_on_it(dim, dtype, nq, nk, at):
    """A NaN in a query row makes that row's output and every dk and dv of its head NaN, one in a key
    every row of the head; the other head stays as it was.  In one pass, split, and over few keys."""
    q, do = _rand((1, 2, nq, dim), dtype, 111), _rand((1, 2, nq, dim), dtype, 112)
    k, v = _rand((1, 2, nk, dim), dtype, 113), _rand((1, 2, nk, dim), dtype, 114)
    clean = dense(q, k, v, do, dim ** -0.5)
    bad = q.clone()
    bad[0, 0, at, 5] = math.nan
    out, lse, dq, dk, dv = dense(bad, k, v, do, dim ** -0.5)
    assert out[0, 0, at].isnan().all() and lse[0, 0, at].isnan() and dq[0, 0, at].isnan().all()
    assert dk[0, 0].isnan().all() and dv[0, 0].isnan().all()
    assert all(t[0, 0].isfinite().any(-1).sum() == nq - 1 for t in (out, dq))
    for got, want in zip((out, lse, dq, dk, dv), clean):
        assert torch.allclose(got[0, 1].double(), want[0, 1].double(), rtol=0, atol=2 * U[dtype])
    bad = k.clone()
    bad[0, 0, at, 5] = math.nan
    got = dense(q, bad, v, do, dim ** -0.5)
    assert all(t[0, 0].isnan().all() for t in got)


def test_a_nan_key_spoils_every_row_at_any_place():
    q, k, v = (_rand((1, 1, 40 + 24 * (i > 0), 64), torch.bfloat16, 115 + i) for i in range(3))
    for at in range(64):
        bad = k.clone()
        bad[0, 0, at] = math.nan
        out, lse = attention.flash_attention_lse(q, bad, v, 0.125)
        assert out.isnan().all() and lse.isnan().all(), at
        assert attention.flash_attention(q, bad, v, 0.125).isnan().all(), at


def test_given_gradient_tensors_count_as_changed():
    """Autograd's check for tensors changed in place sees the gradients that are written into the caller's."""
    q, k, v, do = (_rand((1, 2, 20, 64), torch.float16, 121 + i) for i in range(4))
    out, lse = attention.flash_attention_lse(q, k, v, 0.125)
    fused = torch.zeros((1, 2, 3, 20, 64), dtype=torch.float16, device=DEV)
    before = fused._version
    attention.flash_attention_backward(do.transpose(1, 2).flatten(2), q, k, v, out, lse, 0.125, grads=fused.unbind(2))
    assert fused._version > before


@pytest.mark.parametrize("nq,nk,heads,kv_heads,dim,dtype", [(130, 40000, 2, 1, 64, torch.bfloat16),
                                                            (40000, 130, 2, 2, 128, torch.float16),
                                                            (20011, 20011, 1, 1, 64, torch.float16)])
def test_long_sequences_match_float64(nq, nk, heads, kv_heads, dim, dtype):
    """Streams of hundreds of blocks, split and whole."""
    q, do = _rand((1, heads, nq, dim), dtype, 131), _rand((1, heads, nq, dim), dtype, 132)
    k, v = _rand((1, kv_heads, nk, dim), dtype, 133), _rand((1, kv_heads, nk, dim), dtype, 134)
    compare(q, k, v, do, dim ** -0.5)
