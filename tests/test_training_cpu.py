"""The training operators' refusals and host arithmetic, which need no GPU."""

from __future__ import annotations

import ctypes
import re

import pytest
import torch
from conftest import REPO

from hi3d_b200 import _lib, attention, optim, vae


def _bwd(**kw):
    a = _lib.AttnBwdArgs(*[16] * 9, *[64] * 24, None, None, 5, 7, 1, 2, 2, 64, _lib.F16, 0.125)
    for name, value in kw.items():
        setattr(a, name, value)
    n = ctypes.c_int64(-1)
    return _lib.load().hi3d_flash_attn_bwd_workspace_size(ctypes.byref(a), ctypes.byref(n)), n.value


def test_attention_backward_arguments():
    assert _bwd()[0] == _lib.OK and _bwd()[1] > 0
    for kw in (dict(q=None), dict(lse=None), dict(dk=None), dict(dtype=_lib.F32), dict(nq=0), dict(nk=0),
               dict(num_seqs=0), dict(kv_heads=0), dict(heads=3), dict(q=24), dict(dv_row=60), dict(k_head=-8),
               dict(cu_seqlens_k=16), dict(nq=1 << 31), dict(scale=-1.0), dict(scale=float("nan"))):
        assert _bwd(**kw)[0] == _lib.ERR_INVALID_ARGUMENT, kw
    assert _bwd(head_dim=80)[0] == _lib.ERR_UNSUPPORTED
    a = _lib.AttnBwdArgs(*[16] * 9, *[64] * 24, None, None, 5, 7, 1, 2, 2, 64, _lib.F16, 0.125)
    assert _lib.load().hi3d_flash_attn_bwd(ctypes.byref(a), None, 0, None) == _lib.ERR_CAPACITY
    assert _lib.load().hi3d_flash_attn_bwd(ctypes.byref(a), 256, 64, None) == _lib.ERR_CAPACITY


def test_attention_backward_workspace_covers_a_tile_per_sequence():
    """Packed queries: each sequence's statistics begin at a 128-row tile of their own (8 bytes a row
    and head, in tiles: rows / 128 + sequences of them)."""
    rc, n = _bwd(cu_seqlens_q=16, cu_seqlens_k=16, nq=1000, nk=1000, num_seqs=6)
    assert rc == _lib.OK and n >= (1000 // 128 + 6) * 128 * 8 * 2


def test_attention_forward_lse_arguments():
    lib = _lib.load()
    a = _lib.AttnArgs(q=16, k=16, v=16, out=16, head_dim=64, dtype=0, heads=4, num_seqs=1, nq=1, nk=1)
    call = lambda kv, lse, splits: lib.hi3d_flash_attn_fwd_lse(ctypes.byref(a), kv, lse, splits, None, 0, None)  # noqa: E731
    assert call(3, 16, 1) == _lib.ERR_INVALID_ARGUMENT
    assert call(4, None, 1) == _lib.ERR_INVALID_ARGUMENT
    assert call(4, 16, 65) == _lib.ERR_INVALID_ARGUMENT
    assert call(4, 16, 2) == _lib.ERR_CAPACITY
    a.scale = -0.5
    assert call(4, 16, 1) == _lib.ERR_INVALID_ARGUMENT
    a.scale, a.nk = 0.5, 0
    assert call(4, 16, 1) == _lib.ERR_INVALID_ARGUMENT


def _norm(**kw):
    a = _lib.GroupNormArgs(*[16] * 3, None, *[16] * 7, 10, 64, 1, 8, 1, _lib.F16, 1e-6)
    for name, value in kw.items():
        setattr(a, name, value)
    n = ctypes.c_int64(-1)
    return _lib.load().hi3d_group_norm_act_workspace_size(ctypes.byref(a), ctypes.byref(n)), n.value


def test_group_norm_arguments():
    assert _norm()[0] == _lib.OK and _norm()[1] > 0
    for kw in (dict(rows=-1), dict(samples=0), dict(samples=3), dict(groups=7), dict(groups=0), dict(channels=0),
               dict(dtype=_lib.I32), dict(act=2), dict(eps=0.0), dict(rows=0x7ff00001)):
        assert _norm(**kw)[0] == _lib.ERR_INVALID_ARGUMENT, kw
    for kw in (dict(channels=8192, groups=8192), dict(channels=1 << 21), dict(samples=70000, rows=70000)):
        assert _norm(**kw)[0] == _lib.ERR_UNSUPPORTED, kw
    a = _lib.GroupNormArgs(rows=10, channels=64, samples=1, groups=8, act=1, dtype=_lib.F16, eps=1e-6)
    lib = _lib.load()
    assert lib.hi3d_group_norm_act_fwd(ctypes.byref(a), None, 0, None) == _lib.ERR_INVALID_ARGUMENT
    assert lib.hi3d_group_norm_act_bwd(ctypes.byref(a), None, 0, None) == _lib.ERR_INVALID_ARGUMENT
    a.weight = a.bias = a.mean = a.rstd = a.x = a.y = 16
    assert lib.hi3d_group_norm_act_fwd(ctypes.byref(a), None, 0, None) == _lib.ERR_CAPACITY


def _adamw(numels=(300, 5), offsets=(0, 512), ptrs=(16, 32), **kw):
    n = len(numels)
    a = _lib.AdamWArgs((ctypes.c_void_p * n)(*ptrs), (ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numels),
                       (ctypes.c_int64 * n)(*offsets), None, 16, 16, None, None, 768, 1, 1e-3, 0.9, 0.999, 1e-8, 0.01,
                       n, _lib.F32, 32)
    for name, value in kw.items():
        setattr(a, name, value)
    return _lib.load().hi3d_adamw_step(ctypes.byref(a), None)


def test_adamw_arguments():
    for kw in (dict(step=0), dict(lr=-1.0), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1e-8), dict(weight_decay=-1.0),
               dict(dtype=_lib.I32), dict(dtype=_lib.F16), dict(master=16), dict(state_bits=16), dict(state_bits=8),
               dict(scales=16), dict(exp_avg=None), dict(exp_avg=20), dict(total=700), dict(total=512),
               dict(offsets=(0, 500)), dict(offsets=(0, -256)), dict(offsets=(0, 1024)), dict(numels=(300, -1)),
               dict(ptrs=(16, 30)), dict(ptrs=(16, None)), dict(lr=float("nan"))):
        assert _adamw(**kw) == _lib.ERR_INVALID_ARGUMENT, kw
    assert _adamw(count=0) == _lib.OK
    assert _lib.load().hi3d_adamw_step(None, None) == _lib.ERR_INVALID_ARGUMENT


def test_state_layout_aligns_each_tensor_to_a_block():
    offsets, total = optim.state_layout([1, 256, 257, 0, 5])
    assert offsets == [0, 256, 512, 1024, 1024] and total == 1280
    assert optim.state_layout([]) == ([], 0)


def test_no_cpu_path():
    t = torch.zeros(1, 1, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        attention.flash_attention_lse(t, t, t, 0.1)
    with pytest.raises(ValueError):
        vae.group_norm_act(torch.zeros(4, 8), torch.ones(8), torch.zeros(8), 2)
    with pytest.raises(ValueError):
        optim.adamw_step([torch.zeros(4)], [torch.zeros(4)], torch.zeros(256), torch.zeros(256), step=1, lr=1e-3)


def _statements(src: str, word: str):
    """For each call of `word` in C++ source without comments: its statement, and what opened the blocks
    around it."""
    opened, begin = [], 0
    for i, ch in enumerate(src):
        if ch in "{};":
            if ch == "{":
                opened.append(src[begin:i])
            elif ch == "}" and opened:
                opened.pop()
            begin = i + 1
        elif src.startswith(word, i) and not (src[i - 1].isalnum() or src[i - 1] == "_"):
            yield src[begin:src.index(";", i)], list(opened)


@pytest.mark.parametrize("name", ["attention.cu", "attention_bwd.cu"])
def test_a_whole_warp_leaves_a_wait_together(name):
    """A bounded wait may be given up by some lanes and met by others.  Outside blocks that one lane
    runs, a lane's own result of a wait is not used, neither to leave a loop nor to issue: a vote gives
    the warp one result, or the warp looks at the abort flag after its loop."""
    src = re.sub(r"//[^\n]*", "", (REPO / "hi3dv1.0-mlx_b200" / "csrc" / name).read_text())
    own = [s for s, around in _statements(src, "mbar_wait(") if not any("lane == 0" in b for b in around)]
    for s in own:
        assert re.match(r"\s*(if \([^?]*\) )?mbar_wait\([^;=]*\)$", s), s
    assert own and "if (!__any_sync(0xffffffffu, *abort) && warp_wait(" in src
    # issuing warps that went on after a time-out see their products end
    assert re.search(r"if \(__any_sync\(0xffffffffu, \*abort\)\) \{[^}]*tc_commit\(&bar->drained\[\w+\]\);\s*warp_wait\(&bar->drained", src)
    head = (REPO / "hi3dv1.0-mlx_b200" / "csrc" / "common.cuh").read_text()
    body = head[head.index("bool warp_wait("):]
    assert re.search(r"return __all_sync\(0xffffffffu, ok\);", body[:body.index("\n}")])


@pytest.mark.parametrize("name", ["gemm.cu", "sparse.cu"])
def test_epilogue_warps_leave_a_wait_together(name):
    src = (REPO / "hi3dv1.0-mlx_b200" / "csrc" / name).read_text()
    waits = re.findall(r"(mbar_wait|warp_wait)\(&bar->acc_full", src)
    assert waits and set(waits) == {"warp_wait"}


def test_group_norm_workspace_is_sized_on_the_device_of_x(monkeypatch):
    """The size follows the SM count of the current device, so the device of x has to be the current one."""
    current, asked = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *exc):
            current.pop()

    class Library:
        @staticmethod
        def hi3d_group_norm_act_workspace_size(args, nbytes):
            asked.append(current[-1])
            return _lib.OK

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "load", Library)
    vae._norm_plan.__wrapped__((90, 64), torch.float32, (64,), (64,), 8, "swish", 1e-6, None, (3, 3, 3, 3))
    assert asked == [3] and current == [0]


def test_adamw_tensors_that_share_state_are_refused():
    for numels, offsets in (((300, 5), (0, 256)), ((5, 300), (256, 0)), ((256, 256), (256, 256)), ((1, 256), (0, 0)),
                            ((5, 0, 300), (512, 0, 256))):
        ptrs = tuple(16 * (i + 1) for i in range(len(numels)))
        assert _adamw(numels=numels, offsets=offsets, ptrs=ptrs) == _lib.ERR_INVALID_ARGUMENT, (numels, offsets)
