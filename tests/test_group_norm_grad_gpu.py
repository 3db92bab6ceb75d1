"""Group norm with an activation, and its gradient, against float64.

Tolerances, value by value.  e = 2^-19 (1 + max |mean| / std of the group) covers fp32: a mean of N
std is held to 2^-24 N std, sums of a chunk's rows run in order over at most a few hundred terms,
the sigmoid is good to 2^-21.  y and dx are rounded once to the I/O type (u relative).  dx is the
difference of three terms, so e applies to their sizes; dweight, dbias are sums of N terms, e
applies to the sum of their absolute values.
"""

from __future__ import annotations

import pytest
import torch

from hi3d_b200 import _lib, vae

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-30, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-30}  # half the smallest step


def _rand(shape, seed, dtype=torch.float32):
    return torch.randn(shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)).to(dtype)


def exact(x, dy, w, b, groups, act, lens, eps=1e-6):
    """float64 results and the sizes of their terms, sample by sample, from the formulas."""
    names = ("y", "dx", "size_y", "size_dx", "e")
    got = {n: torch.zeros(x.shape, dtype=torch.float64, device=DEV) for n in names}
    c = x.shape[1]
    dw, db, sw, sb = (torch.zeros(c, dtype=torch.float64, device=DEV) for _ in range(4))
    w, b, at = w.double(), b.double(), 0
    for n in lens:
        s = slice(at, at + n)
        at += n
        if n == 0:
            continue
        t = x[s].double().view(n, groups, -1)
        mean = t.mean((0, 2), keepdim=True)
        std = ((t - mean).square().mean((0, 2), keepdim=True) + eps).sqrt()
        xh = ((t - mean) / std).view(n, c)
        e = (2.0 ** -19 * (1 + mean.abs() / std)).expand(t.shape).reshape(n, c)
        u = xh * w + b
        sig = torch.sigmoid(u) if act else torch.ones_like(u)
        g = sig * (1 + u * (1 - sig)) if act else sig
        du = dy[s].double() * g
        dh = (du * w).view(n, groups, -1)
        c1, c2 = dh.mean((0, 2), keepdim=True), (dh * xh.view(t.shape)).mean((0, 2), keepdim=True)
        dx = (dh - c1 - xh.view(t.shape) * c2) / std
        got["y"][s], got["dx"][s], got["e"][s] = u * sig, dx.view(n, c), e
        got["size_y"][s] = (xh.abs() + 1) * w.abs() + b.abs()
        # the gradient's slope in u is at most about 1.1, so e of u (times |dy|) enters du
        d = dy[s].double().abs() * (1 + (xh.abs() + 1) * w.abs() + b.abs())
        dd = (d * w.abs()).view(n, groups, -1)
        a1, a2 = dd.mean((0, 2), keepdim=True), (dd * (1 + xh.view(t.shape).abs())).mean((0, 2), keepdim=True)
        got["size_dx"][s] = ((dd + a1 + (1 + xh.view(t.shape).abs()) * a2) / std).view(n, c)
        dw, db = dw + (du * xh).sum(0), db + du.sum(0)
        sw, sb = sw + (e * d * (1 + xh.abs())).sum(0), sb + (e * d).sum(0)
    return got, dw, db, sw, sb


def compare(x, dy, w, b, groups, act, lens, packed=True):
    offsets = None
    if packed:
        offsets = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    y, mean, rstd = vae.group_norm_act(x, w, b, groups, act=act, offsets=offsets)
    dx, dw, db = vae.group_norm_act_backward(dy, x, mean, rstd, w, b, act=act, offsets=offsets)
    flat = x.reshape(-1, x.shape[-1])
    t, edw, edb, sw, sb = exact(flat, dy.reshape(flat.shape), w, b, groups, act, lens)
    u = U[x.dtype]
    for name, got in (("y", y), ("dx", dx)):
        err = (got.reshape(flat.shape).double() - t[name]).abs()
        bound = u * t[name].abs() + t["e"] * t["size_" + name] + TINY[x.dtype]
        assert (err <= bound).all(), (name, float((err - bound).max()))
    assert ((dw.double() - edw).abs() <= sw + 1e-12).all()
    assert ((db.double() - edb).abs() <= sb + 1e-12).all()
    return y, mean, rstd, dx, dw, db


# 512, 64, 2112: 16-byte vectors (2112 over several column tiles); 12, 20, 7: one channel at a time
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("channels,groups", [(512, 32), (64, 16), (2112, 32), (12, 3), (20, 1), (7, 7), (256, 1),
                                             (24, 4)])
@pytest.mark.parametrize("act", ["swish", None])
def test_ragged_samples_match_float64(channels, groups, dtype, act):
    lens = [1, 0, 700, 0, 33, 2049, 2, 0]
    x = (_rand((sum(lens), channels), 1) * 2 + _rand((channels,), 2)).to(dtype)
    dy = _rand(x.shape, 3, dtype)
    w, b = _rand((channels,), 4) * 0.5 + 1, _rand((channels,), 5) * 0.3
    _, mean, rstd, *_ = compare(x, dy, w, b, groups, act, lens)
    assert (mean[[1, 3, 7]] == 0).all() and torch.allclose(rstd[[1, 3, 7]], torch.tensor(1e3, device=DEV), rtol=1e-6)


@pytest.mark.parametrize("rows", [1, 2, 31, 40000])
def test_one_sample_and_a_large_mean(rows):
    """A mean of 300 standard deviations: sums about the first value keep the variance's bits."""
    x = _rand((rows, 96), 6) + 300.0
    compare(x, _rand(x.shape, 7), _rand((96,), 8), _rand((96,), 9), 32, "swish", [rows], packed=False)


def test_dense_batches_equal_their_samples():
    x, dy = _rand((3, 5, 41, 64), 10, torch.float16), _rand((3, 5, 41, 64), 11, torch.float16)
    w, b = _rand((64,), 12), _rand((64,), 13)
    y, mean, rstd, dx, dw, db = compare(x, dy, w, b, 8, "swish", [205] * 3, packed=False)
    assert y.shape == x.shape and mean.shape == (3, 8)
    for i in range(3):
        yi, mi, ri = vae.group_norm_act(x[i].reshape(-1, 64), w, b, 8)
        assert torch.allclose(yi.float(), y[i].reshape(-1, 64).float(), rtol=2e-3, atol=1e-4)


def test_forward_agrees_with_the_decoder_norm():
    """The statistics that the decoder's own forward takes (one sample, fp16): equal up to fp32."""
    x = _rand((20000, 256), 14, torch.float16) * 2
    w, b = _rand((256,), 15), _rand((256,), 16)
    mean, inv = vae.group_stats(x)
    want = vae.group_norm_swish(x, mean, inv, w, b)
    y, m, r = vae.group_norm_act(x, w, b, 32)
    assert torch.allclose(m[0].repeat_interleave(8), mean, rtol=1e-4, atol=1e-5)
    assert torch.allclose(r[0].repeat_interleave(8), inv, rtol=1e-5)
    assert ((y.float() - want.float()).abs() <= 2 * U[torch.float16] * want.float().abs() + 1e-4).all()


def test_constant_rows_and_extreme_values():
    x = torch.full((100, 32), 5.0, device=DEV)
    y, mean, rstd = vae.group_norm_act(x, torch.ones(32, device=DEV), torch.zeros(32, device=DEV), 4)
    assert not y.any() and (mean == 5).all() and torch.allclose(rstd, torch.tensor(1e3, device=DEV), rtol=1e-6)
    x = _rand((500, 32), 17)
    w, b = torch.full((32,), 200.0, device=DEV), torch.zeros(32, device=DEV)  # u from -700 to 700
    y, mean, rstd = vae.group_norm_act(x, w, b, 4)
    dx, dw, db = vae.group_norm_act_backward(torch.ones_like(x), x, mean, rstd, w, b)
    assert all(torch.isfinite(t).all() for t in (y, dx, dw, db)) and (y[y < 0] >= -0.3).all()


def test_a_sample_of_nan_or_infinities_stays_alone():
    lens = [100, 60, 200]
    x, dy = _rand((360, 64), 18, torch.float16), _rand((360, 64), 19, torch.float16)
    w, b = _rand((64,), 20), _rand((64,), 21)
    offsets = torch.tensor([0, 100, 160, 360], dtype=torch.int32, device=DEV)
    clean = vae.group_norm_act(x, w, b, 8, offsets=offsets)
    cdx = vae.group_norm_act_backward(dy, x, *clean[1:], w, b, offsets=offsets)[0]
    x[100:160] = float("nan")
    x[120] = float("inf")
    y, mean, rstd = vae.group_norm_act(x, w, b, 8, offsets=offsets)
    dx = vae.group_norm_act_backward(dy, x, mean, rstd, w, b, offsets=offsets)[0]
    keep = torch.cat([torch.arange(100), torch.arange(160, 360)]).to(DEV)
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], cdx[keep])
    assert torch.isnan(y[100:160]).all()


def test_gradients_match_differences():
    """Central differences of the float64 norm along a random direction (step 1e-5: truncation
    1e-10, rounding 1e-11 relative) against <gradient, direction>: e over the terms' sizes."""
    lens = [40, 9]
    x, dy, w, b = _rand((49, 24), 22), _rand((49, 24), 23), _rand((24,), 24) + 1, _rand((24,), 25)
    _, _, _, dx, dw, db = compare(x, dy, w, b, 4, "swish", lens)
    step = [_rand(t.shape, 26 + i).double() for i, t in enumerate((x, w, b))]

    def f(h):
        y = exact(x.double() + h * step[0], dy, w.double() + h * step[1], b.double() + h * step[2], 4, True, lens)[0]["y"]
        return (y * dy.double()).sum()

    diff = (f(1e-5) - f(-1e-5)) / 2e-5
    got = sum((g.double() * s).sum() for g, s in zip((dx, dw, db), step))
    t, *_, sw, sb = exact(x, dy, w, b, 4, True, lens)
    bound = ((t["e"] * t["size_dx"] + U[torch.float32] * t["dx"].abs()) * step[0].abs()).sum()
    bound = bound + (sw * step[1].abs()).sum() + (sb * step[2].abs()).sum()
    assert abs(got - diff) <= bound + 1e-6 * abs(diff)


def test_strides_alignment_streams_and_determinism():
    wide = _rand((333, 3, 64), 30, torch.bfloat16)
    x, dy = wide[:, 1], wide[:, 2]
    odd = torch.empty(333 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(333, 64)
    odd.copy_(x)
    w, b = _rand((64,), 31), _rand((64,), 32)
    want = vae.group_norm_act(x, w, b, 8)
    want += vae.group_norm_act_backward(dy, x, *want[1:], w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = vae.group_norm_act(x, w, b, 8)
        again += vae.group_norm_act_backward(dy, x, *again[1:], w, b)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, again))
    compare(odd, dy.contiguous(), w, b, 8, "swish", [333], packed=False)  # 2 bytes past an aligned address


def test_element_offsets_past_31_bits():
    """2^31 elements and more, the last rows checked: one sample's statistics are known."""
    rows, c = (1 << 31) // 64 + 4097, 64
    x = torch.empty((rows, c), dtype=torch.float16, device=DEV)
    x[0::2], x[1::2] = 1.0, 3.0  # mean 2, variance 1 up to one row
    w, b = torch.ones(c, device=DEV), torch.zeros(c, device=DEV)
    y, mean, rstd = vae.group_norm_act(x, w, b, 32, act=None)
    assert torch.allclose(mean, torch.tensor(2.0, device=DEV), rtol=1e-5)
    assert torch.allclose(rstd, torch.tensor(1.0, device=DEV), rtol=1e-5)
    assert torch.allclose(y[-5000:].float().abs(), torch.tensor(1.0, device=DEV), rtol=1e-3)
    dx, dw, db = vae.group_norm_act_backward(y, x, mean, rstd, w, b, act=None)
    # dy = xh: dw = sum xh^2 = rows, db = 0 up to one row, dx = 0
    assert torch.allclose(dw, torch.tensor(float(rows), device=DEV), rtol=1e-3) and (db.abs() < 0.01 * rows).all()
    assert dx[-5000:].abs().max() < 1e-2


def test_no_rows():
    x = torch.empty((0, 16), device=DEV)
    w, b = torch.ones(16, device=DEV), torch.zeros(16, device=DEV)
    offsets = torch.zeros(3, dtype=torch.int32, device=DEV)
    y, mean, rstd = vae.group_norm_act(x, w, b, 4, offsets=offsets)
    dx, dw, db = vae.group_norm_act_backward(y, x, mean, rstd, w, b, offsets=offsets)
    assert y.shape == (0, 16) and (mean == 0).all() and not dw.any() and not db.any()
    y, mean, _ = vae.group_norm_act(torch.empty((0, 5, 16), device=DEV), w, b, 4)
    assert y.shape == (0, 5, 16) and mean.shape == (0, 4)
    assert _lib.device_status()["code"] == 0


def test_refusals():
    x, w, b = _rand((9, 16), 40), _rand((16,), 41), _rand((16,), 42)
    with pytest.raises(ValueError):
        vae.group_norm_act(x.double(), w, b, 4)
    with pytest.raises(ValueError):
        vae.group_norm_act(x, w, b, 5)
    with pytest.raises(ValueError):
        vae.group_norm_act(x, w[:8], b, 4)
    with pytest.raises(ValueError):
        vae.group_norm_act(x, w, b, 4, act="gelu")
    with pytest.raises(ValueError):
        vae.group_norm_act(x, w, b, 4, eps=0.0)
    with pytest.raises(ValueError):
        vae.group_norm_act(x.cpu(), w, b, 4)
    with pytest.raises(ValueError):
        vae.group_norm_act(x[None], w, b, 4, offsets=torch.tensor([0, 9], dtype=torch.int32, device=DEV))
    y, mean, rstd = vae.group_norm_act(x, w, b, 4)
    with pytest.raises(ValueError):
        vae.group_norm_act_backward(y.half(), x, mean, rstd, w, b)
    with pytest.raises(ValueError):
        vae.group_norm_act_backward(y, x, mean.expand(2, 4), rstd.expand(2, 4), w, b)


@pytest.mark.parametrize("first", [0.0, 30.0, -3000.0])
@pytest.mark.parametrize("mean", [0.0, 300.0])
@pytest.mark.parametrize("samples,rows,channels", [(140, 677, 1024), (1, 40000, 64)])
def test_an_atypical_first_row_costs_no_bits(first, mean, samples, rows, channels):
    """A first row far from the others, in samples whose hundreds of rows one thread sums and in one of
    many chunks: the same bounds."""
    x = _rand((samples, rows, channels), 50) + mean
    x[:, 0] = first
    compare(x, _rand(x.shape, 51), _rand((channels,), 52) * 0.5 + 1, _rand((channels,), 53), 32, "swish",
            [rows] * samples, packed=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_atypical_first_rows_of_many_chunks(dtype):
    """The first rows, about one chunk of a few hundred, at 1000 where the others are around 0."""
    x = _rand((60000, 64), 54)
    x[:200] += 1000.0
    x = x.to(dtype)
    compare(x, _rand(x.shape, 55, dtype), _rand((64,), 56) * 0.5 + 1, _rand((64,), 57), 32, "swish", [60000],
            packed=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("channels", [32, 7])
def test_swish_far_from_zero(dtype, channels):
    """u sigmoid(u) of a very negative u is 0 and so is its slope (both below 1e-15 from -40 on); a large u
    passes with slope 1, whatever its neighbour channel holds."""
    x, dy = _rand((200, channels), 60, dtype), _rand((200, channels), 61, dtype)
    w = torch.ones(channels, device=DEV)
    b = torch.tensor([1e6, 0.3, -1e20, -0.5, -1e4, 1e20, 50.0], device=DEV).repeat(5)[:channels]
    y, mean, rstd = vae.group_norm_act(x, w, b, 1)
    dx, dw, db = vae.group_norm_act_backward(dy, x, mean, rstd, w, b)
    low, high = b < -1000, b > 1000
    assert (y[:, low].abs() <= 1e-15).all() and (db[low].abs() <= 1e-12).all() and (dw[low].abs() <= 1e-12).all()
    assert torch.allclose(y[:, high].double(), b[high].double().expand_as(y[:, high]), rtol=2 * U[dtype] + 1e-5)
    size = dy.double().abs().sum(0)
    assert ((db.double() - dy.double().sum(0)).abs()[high] <= 1e-6 * size[high]).all()
    assert torch.isfinite(dx).all()
