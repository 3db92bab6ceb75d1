"""Cases of the training operators: attention with its gradient, group norm with an activation and its gradient,
and the AdamW step, each in its plain form and through hi3d_b200."""

import itertools
import math
import sys

import torch

own = False  # False: the plain form; True: the framework's operators

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 256  # elements per 8-bit scale, and the alignment of a tensor in the flat optimizer state


def listed():
    return [
        # a short conditioning prompt attended by a small crop: launch latency counts
        {"name": "attn_cross_small_f16", "op": "attention", "form": "dense", "dtype": "f16", "batch": 1, "heads": 4,
         "kv_heads": 4, "dim": 64, "nq": 512, "nk": 77, "shared": False},
        # self-attention of one block over the 4,096-voxel shell
        {"name": "attn_self_4096_bf16", "op": "attention", "form": "dense", "dtype": "bf16", "batch": 1, "heads": 16,
         "kv_heads": 16, "dim": 64, "nq": 4096, "nk": 4096, "shared": False},
        # two branches attending one set of image-encoder tokens: the K/V gradient sums over the batch
        {"name": "attn_cross_shared_bf16", "op": "attention", "form": "dense", "dtype": "bf16", "batch": 2,
         "heads": 16, "kv_heads": 16, "dim": 64, "nq": 4096, "nk": 1370, "shared": True},
        # a packed batch of ragged objects at the released head layout, one of them empty, one a single voxel
        {"name": "attn_packed_ragged_f16", "op": "attention", "form": "packed", "dtype": "f16", "heads": 22,
         "kv_heads": 22, "dim": 96, "lens_q": "1733,0,2048,1,1091", "lens_k": "1733,0,2048,1,1091"},
        # few wide heads with grouped keys, an odd length
        {"name": "attn_grouped_2049_bf16", "op": "attention", "form": "dense", "dtype": "bf16", "batch": 1,
         "heads": 16, "kv_heads": 4, "dim": 128, "nq": 2049, "nk": 2049, "shared": False},
        # the longest self-attention whose plain form fits beside its inputs
        {"name": "attn_self_8192_bf16", "op": "attention", "form": "dense", "dtype": "bf16", "batch": 1, "heads": 16,
         "kv_heads": 16, "dim": 64, "nq": 8192, "nk": 8192, "shared": False},
        # a residual block's norm on a few hundred voxels
        {"name": "norm_small_f16", "op": "norm", "dtype": "f16", "lens": "512", "channels": 256, "groups": 32,
         "swish": True},
        # a ragged batch of objects, one of them empty
        {"name": "norm_ragged_bf16", "op": "norm", "dtype": "bf16", "lens": "40961,0,3,25000,34036", "channels": 512,
         "groups": 32, "swish": True},
        # the decoder's finest level: 200,000 voxels
        {"name": "norm_200k_f32", "op": "norm", "dtype": "f32", "lens": "200000", "channels": 256, "groups": 32,
         "swish": True},
        # a fine-tuned head: few small tensors
        {"name": "adamw_small_f32", "op": "adamw", "dtype": "f32", "blocks": 1, "width": 96, "bits": 32},
        # four 1024-wide blocks, 16-bit weights with 32-bit masters
        {"name": "adamw_blocks_bf16", "op": "adamw", "dtype": "bf16", "blocks": 4, "width": 1024, "bits": 32},
        # the 24-block stack with 8-bit states
        {"name": "adamw_stack_8bit_bf16", "op": "adamw", "dtype": "bf16", "blocks": 24, "width": 1024, "bits": 8},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm", "adamw"])
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8, 11, 16, 22])
        group = rng.choice([1, 1, 1, 2, 4]) if kv_heads <= 8 else 1
        case = {"op": op, "form": rng.choice(["dense", "dense", "packed"]), "dtype": rng.choice(["f16", "bf16"]),
                "heads": kv_heads * group, "kv_heads": kv_heads, "dim": rng.choice([64, 64, 96, 128])}
        if case["form"] == "dense":
            batch = rng.choice([1, 1, 2, 3])
            case |= {"batch": batch, "nq": _spread(rng, 1, 6000), "nk": _spread(rng, 2, 6000),
                     "shared": batch > 1 and rng.random() < 0.5}
            if rng.random() < 0.4:
                case["nq"] = case["nk"]
        else:
            n = rng.choice([2, 3, 4, 6])
            lens = [rng.choice([0, 1, _spread(rng, 2, 2500), _spread(rng, 100, 2500)]) for _ in range(n)]
            lens[rng.randrange(n)] = _spread(rng, 100, 2500)
            other = lens if rng.random() < 0.6 else [rng.choice([0, _spread(rng, 1, 2500)]) for _ in range(n - 1)] + [77]
            case |= {"lens_q": ",".join(map(str, lens)), "lens_k": ",".join(map(str, other))}
        if work(case)["flops"] > 4e11 or _padded(case) > 4e8:
            return draw(rng)
        return case
    if op == "norm":
        groups = rng.choice([1, 4, 8, 16, 32])
        channels = groups * rng.choice([1, 2, 3, 4, 6, 8, 16])
        n = rng.choice([1, 1, 2, 3, 5])
        rows = min(200000, 25_000_000 // channels)
        lens = [_spread(rng, 1, max(1, rows // n)) if rng.random() < 0.9 else 0 for _ in range(n)]
        lens[0] = max(lens[0], _spread(rng, 1000, 4000))
        return {"op": op, "dtype": rng.choice(["f16", "bf16", "f32"]), "lens": ",".join(map(str, lens)),
                "channels": channels, "groups": groups, "swish": rng.random() < 0.8}
    return {"op": op, "dtype": rng.choice(["f16", "bf16", "f32"]), "blocks": rng.choice([1, 2, 3, 5]),
            "width": 2 * _spread(rng, 20, 450) + 1, "bits": rng.choice([8, 32])}


def _ints(text):
    return [int(t) for t in text.split(",")]


def _offsets(lens, device="cuda"):
    return torch.tensor(list(itertools.accumulate(lens, initial=0)), dtype=torch.int32, device=device)


def _padded(case):
    """Scores that the plain form holds at once."""
    if case["form"] == "dense":
        return case["batch"] * case["heads"] * case["nq"] * case["nk"]
    lq, lk = _ints(case["lens_q"]), _ints(case["lens_k"])
    return len(lq) * case["heads"] * max(lq) * max(lk)


def _block_shapes(case):
    """The tensors of `blocks` transformer blocks: attention, cross-attention and MLP weights, biases, norms, gains."""
    c = case["width"]
    one = [(6 * c,), (3 * c, c), (3 * c,), (c,), (c,), (c, c), (c,), (c,), (c,), (c, c), (c,), (2 * c, c), (2 * c,),
           (c, c), (c,), (4 * c, c), (4 * c,), (c, 4 * c), (c,)]
    return one * case["blocks"]


def _places(shapes):
    """(offset, elements) of each tensor in a flat buffer whose tensors begin at multiples of BLOCK, and its length."""
    sizes = [math.prod(s) for s in shapes]
    at = list(itertools.accumulate((-(-n // BLOCK) * BLOCK for n in sizes), initial=0))
    return list(zip(at, sizes)), at[-1]


def work(case):
    if case["op"] == "attention":
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        if case["form"] == "dense":
            b, bk = case["batch"], 1 if case["shared"] else case["batch"]
            rows, keys, pairs = b * case["nq"], bk * case["nk"], b * case["nq"] * case["nk"]
        else:
            lq, lk = _ints(case["lens_q"]), _ints(case["lens_k"])
            rows, keys, pairs = sum(lq), sum(lk), sum(x * y for x, y in zip(lq, lk))
        # q, dout read, out, dq written; k, v read, dk, dv written; the log-sum-exp written.  Two products forward,
        # five backward.
        return {"bytes": 2 * (4 * rows * h * d + 4 * keys * hk * d) + 4 * rows * h, "flops": 14 * pairs * h * d}
    if case["op"] == "norm":
        n = sum(_ints(case["lens"])) * case["channels"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 4 * n * size + 16 * case["channels"], "flops": 30 * n}
    n = sum(k for _, k in _places(_block_shapes(case))[0])
    # 12: in 32 bits the weight read and written and the gradient; in 16 the gradient, the weight written, the master
    # read and written.  Both states read and written in 4 bytes each, or in one with two scales a block.
    return {"bytes": n * (12 + (4 + 16 / BLOCK if case["bits"] == 8 else 16)), "flops": 15 * n}


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    norm = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    if case["op"] == "attention":
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        # queries and keys as they leave the QK norm (unit variance), values of a projection, a loss's gradient
        if case["form"] == "dense":
            b, bk, nq, nk = case["batch"], 1 if case["shared"] else case["batch"], case["nq"], case["nk"]
            q, k, v = norm(b, h, nq, d).to(dt), norm(bk, hk, nk, d).to(dt), norm(bk, hk, nk, d).to(dt)
            return {"case": case, "q": q, "k": k, "v": v, "dout": (norm(b, nq, h * d) * 0.1).to(dt)}
        lq, lk = _ints(case["lens_q"]), _ints(case["lens_k"])
        if lq == lk and h == hk:  # self-attention: views of one fused projection
            q, k, v = norm(sum(lq), 3, h, d).to(dt).unbind(1)
        else:
            q = norm(sum(lq), h, d).to(dt)
            k, v = norm(sum(lk), 2, hk, d).to(dt).unbind(1)
        return {"case": case, "q": q, "k": k, "v": v, "dout": (norm(sum(lq), h, d) * 0.1).to(dt),
                "cu_q": _offsets(lq), "cu_k": _offsets(lk), "max_q": max(lq), "max_k": max(lk)}
    if case["op"] == "norm":
        c, lens = case["channels"], _ints(case["lens"])
        # features with a spread and an offset of their own per channel
        x = norm(sum(lens), c) * (0.5 + 2.5 * torch.rand(c, device="cuda", generator=g)) + norm(c)
        w, b = 0.5 + torch.rand(c, device="cuda", generator=g), 0.2 * norm(c)
        return {"case": case, "x": x.to(dt), "dy": (norm(sum(lens), c) * 0.1).to(dt), "w": w, "b": b, "lens": lens,
                "offsets": _offsets(lens) if len(lens) > 1 else None}
    shapes = _block_shapes(case)
    places, total = _places(shapes)
    keep = torch.zeros(total, dtype=torch.bool, device="cuda")
    keep[torch.cat([torch.arange(at, at + n, device="cuda") for at, n in places])] = True
    flat = lambda t: t.masked_fill_(~keep, 0)  # noqa: E731
    views = lambda t: [t[at:at + n].view(s) for (at, n), s in zip(places, shapes)]  # noqa: E731
    master = flat(norm(total).mul_(0.02))
    m, u = flat(norm(total).mul_(1e-3)), flat(norm(total).abs_().mul_(1e-3).add_(1e-5))
    grad = flat(norm(total).mul_(1e-3)).to(dt)
    state = {"case": case, "param": master.to(dt) if dt != torch.float32 else master,
             "master": None if dt == torch.float32 else master, "step": 10}
    if case["bits"] == 8:
        state["scales"] = torch.stack([m.view(-1, BLOCK).abs().amax(1), u.view(-1, BLOCK).amax(1)]) / 448
        code = lambda t, s: (t.view(-1, BLOCK) / s.clamp_min(1e-30)[:, None]).to(torch.float8_e4m3fn).view(-1)  # noqa: E731
        state["m"], state["v"] = code(m, state["scales"][0]), code(u, state["scales"][1])
    else:
        state["m"], state["v"] = m, u.square_()
    state["params"], state["grads"] = views(state["param"]), views(grad)
    return state


def run(s):
    op = s["case"]["op"]
    if op == "attention":
        return _attention_own(s) if own else _attention(s)
    if op == "norm":
        return _norm_own(s) if own else _norm(s)
    s["step"] += 1
    if own:
        _adamw_own(s)
    elif s["case"]["bits"] == 8:
        _adamw8(s)
    else:
        _adamw(s)
    out = {"param": s["param"], "exp_avg": s["m"], "exp_avg_sq": s["v"]}
    if s["master"] is not None:
        out["master"] = s["master"]
    if s["case"]["bits"] == 8:
        out["scales"] = s["scales"]
    return out


HYPER = {"lr": 1e-4, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}


# ---------------------------------------------------------------- through the framework
def _package():
    if "hi3dv1.0-mlx_b200" not in sys.path:
        sys.path.insert(1, "hi3dv1.0-mlx_b200")
    import hi3d_b200

    return hi3d_b200


def _attention_own(s):
    _package()
    from hi3d_b200 import attention as at

    scale = s["case"]["dim"] ** -0.5
    if s["case"]["form"] == "dense":
        out, lse = at.flash_attention_lse(s["q"], s["k"], s["v"], scale)
        dq, dk, dv = at.flash_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, scale)
    else:
        out, lse = at.flash_attn_varlen_lse(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["max_q"], scale)
        dq, dk, dv = at.flash_attn_varlen_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, s["cu_q"], s["cu_k"],
                                                   scale)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _norm_own(s):
    _package()
    from hi3d_b200 import vae

    act = "swish" if s["case"]["swish"] else None
    y, mean, rstd = vae.group_norm_act(s["x"], s["w"], s["b"], s["case"]["groups"], act=act, offsets=s["offsets"])
    dx, dw, db = vae.group_norm_act_backward(s["dy"], s["x"], mean, rstd, s["w"], s["b"], act=act,
                                             offsets=s["offsets"])
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _adamw_own(s):
    _package()
    from hi3d_b200 import optim

    optim.adamw_step(s["params"], s["grads"], s["m"], s["v"], step=s["step"], master=s["master"],
                     scales=s.get("scales"), **HYPER)


# ---------------------------------------------------------------- plain forms
def _attend(q, k, v, dout, scale, mask=None):
    """q, dout [B, Hk, G, Nq, D]; k, v [B or 1, Hk, 1, Nk, D]; mask [B, 1, 1, Nq, Nk].  32 bits throughout."""
    s = (q @ k.mT).mul_(scale)
    if mask is not None:
        s.masked_fill_(~mask, float("-inf"))
    top = s.amax(-1, keepdim=True).clamp_min(-3e38)
    p = s.sub_(top).exp_()
    l = p.sum(-1, keepdim=True)
    lse = (top + l.log()).squeeze(-1)
    p.div_(l.clamp_min(1e-38))
    out = p @ v
    dv = (p.mT @ dout).sum(2, keepdim=True)
    dp = dout @ v.mT
    ds = dp.sub_((dout * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = ds @ k
    dk = (ds.mT @ q).sum(2, keepdim=True)
    if k.shape[0] != q.shape[0]:
        dk, dv = dk.sum(0, keepdim=True), dv.sum(0, keepdim=True)
    return out, lse, dq, dk, dv


def _attention(s):
    c = s["case"]
    h, hk, d, dt = c["heads"], c["kv_heads"], c["dim"], s["q"].dtype
    scale = d ** -0.5
    if c["form"] == "dense":
        b, nq = c["batch"], c["nq"]
        q = s["q"].float().view(b, hk, h // hk, nq, d)
        do = s["dout"].float().view(b, nq, hk, h // hk, d).permute(0, 2, 3, 1, 4)
        out, lse, dq, dk, dv = _attend(q, s["k"].float().unsqueeze(2), s["v"].float().unsqueeze(2), do, scale)
        return {"out": out.permute(0, 3, 1, 2, 4).reshape(b, nq, h * d).to(dt), "lse": lse.reshape(b, h, nq),
                "dq": dq.reshape(b, h, nq, d).to(dt), "dk": dk.squeeze(2).to(dt), "dv": dv.squeeze(2).to(dt)}
    # packed: the sequences side by side, padded to the longest
    nq, nk = s["max_q"], max(1, s["max_k"])
    iq = torch.arange(nq, device="cuda")
    ik = torch.arange(nk, device="cuda")
    cq, ck = s["cu_q"].long(), s["cu_k"].long()
    at_q, at_k = cq[:-1, None] + iq, ck[:-1, None] + ik  # [S, N]
    has_q, has_k = at_q < cq[1:, None], at_k < ck[1:, None]
    side = lambda t, at, has: (t[at.clamp_max(t.shape[0] - 1)].float() * has[..., None, None]).permute(0, 2, 1, 3)  # noqa: E731
    n = cq.numel() - 1
    q = side(s["q"], at_q, has_q).reshape(n, hk, h // hk, nq, d)
    do = side(s["dout"], at_q, has_q).reshape(n, hk, h // hk, nq, d)
    k, v = side(s["k"], at_k, has_k).unsqueeze(2), side(s["v"], at_k, has_k).unsqueeze(2)
    mask = (has_q[:, :, None] & has_k[:, None, :])[:, None, None]
    out, lse, dq, dk, dv = _attend(q, k, v, do, scale, mask)
    tq, tk = torch.arange(s["q"].shape[0], device="cuda"), torch.arange(s["k"].shape[0], device="cuda")
    seq_q = (tq[:, None] >= cq[None, 1:]).sum(1)
    seq_k = (tk[:, None] >= ck[None, 1:]).sum(1)
    pos_q, pos_k = tq - cq[seq_q], tk - ck[seq_k]
    rows = lambda t, heads: t.reshape(n, heads, -1, d)  # noqa: E731
    return {"out": rows(out, h)[seq_q, :, pos_q].to(dt), "lse": lse.reshape(n, h, nq)[seq_q, :, pos_q].t().contiguous(),
            "dq": rows(dq, h)[seq_q, :, pos_q].to(dt), "dk": rows(dk, hk)[seq_k, :, pos_k].to(dt),
            "dv": rows(dv, hk)[seq_k, :, pos_k].to(dt)}


def _norm_sample(x, dy, w, b, groups, swish, eps=1e-6):
    """One object: y, dx and its part of the weight and bias gradients."""
    n, c = x.shape
    v = x.float().view(n, groups, -1)
    xc = v - v.mean((0, 2), keepdim=True)
    rstd = xc.square().mean((0, 2), keepdim=True).add_(eps).rsqrt_()
    xh = xc * rstd
    u = (xh.view(n, c) * w + b)
    du = dy.float()
    y = u
    if swish:
        sg = torch.sigmoid(u)
        y = u * sg
        du = du * (sg * (1 + u * (1 - sg)))
    dw, db = (du * xh.view(n, c)).sum(0), du.sum(0)
    dh = (du * w).view(n, groups, -1)
    dx = rstd * (dh - dh.mean((0, 2), keepdim=True) - xh * (dh * xh).mean((0, 2), keepdim=True))
    return y.to(x.dtype), dx.view(n, c).to(x.dtype), dw, db


def _norm(s):
    c = s["case"]
    got = [_norm_sample(x, dy, s["w"], s["b"], c["groups"], c["swish"])
           for x, dy in zip(s["x"].split(s["lens"]), s["dy"].split(s["lens"])) if x.shape[0]]
    y, dx, dw, db = zip(*got)
    return {"y": torch.cat(y), "dx": torch.cat(dx), "dweight": sum(dw), "dbias": sum(db)}


def _moments(s, g, m, v):
    """m and v after this gradient and the step that they ask for, in 32 bits; m and v are changed in place."""
    b1, b2 = HYPER["betas"]
    torch._foreach_mul_(m, b1)
    torch._foreach_add_(m, torch._foreach_mul(g, 1 - b1))
    torch._foreach_mul_(v, b2)
    torch._foreach_mul_(g, g)
    torch._foreach_mul_(g, 1 - b2)
    torch._foreach_add_(v, g)
    den = torch._foreach_sqrt(v)
    torch._foreach_mul_(den, (1 - b2 ** s["step"]) ** -0.5)
    torch._foreach_add_(den, HYPER["eps"])
    up = torch._foreach_div(m, den)
    torch._foreach_mul_(up, HYPER["lr"] / (1 - b1 ** s["step"]))
    return up


def _apply(s, p32, up):
    torch._foreach_mul_(p32, 1 - HYPER["lr"] * HYPER["weight_decay"])
    torch._foreach_sub_(p32, up)
    if s["master"] is not None:
        torch._foreach_copy_(s["params"], p32)


def _views(s, flat):
    places, _ = _places([tuple(p.shape) for p in s["params"]])
    return [flat[at:at + n].view(p.shape) for (at, n), p in zip(places, s["params"])]


def _adamw(s):
    g = [t.float() for t in s["grads"]] if s["master"] is not None else torch._foreach_mul(s["grads"], 1.0)
    up = _moments(s, g, _views(s, s["m"]), _views(s, s["v"]))
    _apply(s, s["params"] if s["master"] is None else _views(s, s["master"]), up)


def _adamw8(s):
    """States in blocks of BLOCK values: an 8-bit float each for m and for the root of v, and the block's scale."""
    m = (s["m"].float().view(-1, BLOCK) * s["scales"][0][:, None]).view(-1)
    u = (s["v"].float().view(-1, BLOCK) * s["scales"][1][:, None]).view(-1)
    v = u * u
    g = [t.float() for t in s["grads"]] if s["master"] is not None else torch._foreach_mul(s["grads"], 1.0)
    up = _moments(s, g, _views(s, m), _views(s, v))
    _apply(s, s["params"] if s["master"] is None else _views(s, s["master"]), up)
    u = v.sqrt_()
    for_m, for_u = m.view(-1, BLOCK), u.view(-1, BLOCK)
    scales = torch.stack([for_m.abs().amax(1), for_u.amax(1)]) * (1 / 448)
    inv = torch.where(scales >= 2.0 ** -120, scales.reciprocal(), 0.0)
    cu = for_u * inv[1][:, None]
    cu = torch.where((for_u > 0) & (inv[1][:, None] > 0), cu.clamp_min(2.0 ** -9), 0.0)
    s["m"].copy_((for_m * inv[0][:, None]).view(-1).to(torch.float8_e4m3fn))
    s["v"].copy_(cu.view(-1).to(torch.float8_e4m3fn))
    s["scales"].copy_(scales)


# ---------------------------------------------------------------- 64 bits, from the definitions
def _exact_attention(q, k, v, do, scale):
    """q, do [Nq, D], k, v [Nk, D] of one head, by autograd on softmax(q k^T scale) v."""
    q, k, v = (t.double().requires_grad_() for t in (q, k, v))
    with torch.enable_grad():
        s = torch.einsum("id,jd->ij", q, k) * scale
        o = torch.einsum("ij,jd->id", torch.softmax(s, -1), v)
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), do.double())
    return o.detach(), torch.logsumexp(s.detach(), -1), dq, dk, dv


def exact(case, seed):
    s = prepare(case, seed)
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    if case["op"] == "attention":
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        dense = case["form"] == "dense"
        out, dq, dk, dv = z(s["dout"]), z(s["q"]), z(s["k"]), z(s["v"])
        if dense:
            lse = torch.zeros(case["batch"], h, case["nq"], dtype=torch.float64, device="cuda")
            do = s["dout"].view(case["batch"], case["nq"], h, d)
            o4 = out.view(case["batch"], case["nq"], h, d)
            for b in range(case["batch"]):
                for i in range(h):
                    j, e = i // (h // hk), 0 if case["shared"] else b
                    r = _exact_attention(s["q"][b, i], s["k"][e, j], s["v"][e, j], do[b, :, i], d ** -0.5)
                    o4[b, :, i], lse[b, i], dq[b, i] = r[:3]
                    dk[e, j] += r[3]
                    dv[e, j] += r[4]
        else:
            lse = torch.full((h, s["q"].shape[0]), float("-inf"), dtype=torch.float64, device="cuda")
            cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
            for n in range(len(cq) - 1):
                a, b, e, f = cq[n], cq[n + 1], ck[n], ck[n + 1]
                for i in range(h if b > a and f > e else 0):
                    j = i // (h // hk)
                    r = _exact_attention(s["q"][a:b, i], s["k"][e:f, j], s["v"][e:f, j], s["dout"][a:b, i], d ** -0.5)
                    out[a:b, i], lse[i, a:b], dq[a:b, i] = r[:3]
                    dk[e:f, j] += r[3]
                    dv[e:f, j] += r[4]
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if case["op"] == "norm":
        w, b = s["w"].double().requires_grad_(), s["b"].double().requires_grad_()
        ys, dxs, dw, db = [], [], 0, 0
        for x, dy in zip(s["x"].split(s["lens"]), s["dy"].split(s["lens"])):
            if not x.shape[0]:
                continue
            with torch.enable_grad():
                x = x.double().requires_grad_()
                t = x.unflatten(1, (case["groups"], -1))
                var, mean = torch.var_mean(t, (0, 2), correction=0, keepdim=True)
                u = ((t - mean) / torch.sqrt(var + 1e-6)).flatten(1) * w + b
                y = u / (1 + torch.exp(-u)) if case["swish"] else u
                gx, gw, gb = torch.autograd.grad(y, (x, w, b), dy.double())
            ys.append(y.detach())
            dxs.append(gx)
            dw, db = dw + gw, db + gb
        return {"y": torch.cat(ys), "dx": torch.cat(dxs), "dweight": dw, "dbias": db}
    eight = case["bits"] == 8
    n, t = s["param"].numel(), s["step"] + 1
    (b1, b2), lr = HYPER["betas"], HYPER["lr"]
    g = torch.zeros(n, dtype=torch.float64, device="cuda")
    for (at, k), x in zip(_places(_block_shapes(case))[0], s["grads"]):
        g[at:at + k] = x.reshape(-1).double()
    p = (s["param"] if s["master"] is None else s["master"]).double()
    m, v = s["m"].double(), s["v"].double()
    if eight:
        m = (m.view(-1, BLOCK) * s["scales"][0][:, None].double()).view(-1)
        v = (v.view(-1, BLOCK) * s["scales"][1][:, None].double()).view(-1).square()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    p = p - lr * HYPER["weight_decay"] * p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + HYPER["eps"])
    out = {"param": p, "exp_avg": m, "exp_avg_sq": v}
    if s["master"] is not None:
        out["master"] = p
    if eight:
        a, c = m.view(-1, BLOCK).abs().amax(1) / 448, v.sqrt().view(-1, BLOCK).amax(1) / 448
        out["scales"] = torch.stack([a, c])
        out["exp_avg"] = (m.view(-1, BLOCK) / a[:, None].clamp_min(1e-300)).to(torch.float8_e4m3fn).double().view(-1)
        r = v.sqrt().view(-1, BLOCK) / c[:, None].clamp_min(1e-300)
        out["exp_avg_sq"] = torch.where(r > 0, r.clamp_min(2.0 ** -9), r).to(torch.float8_e4m3fn).double().view(-1)
    return out
