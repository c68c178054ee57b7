"""Refusals of the norm and int4 product entry points: decided on the host, before any CUDA call, so they run without a
GPU.  Pointers are never followed here."""
import ctypes

import pytest
import torch

FAKE = 1 << 20          # 16-byte and 256-byte aligned stand-in for a device pointer

F32, BF16, F16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    from forge import _abi
    return _abi.load_library()


def _linear(lib, x=FAKE, ldx=64, dtype=BF16, w=FAKE, s=FAKE, gs=32, T=2, C=64, R=16, bias=None, act=0, res=None, ldres=0,
            y=FAKE, z=None):
    return lib.forge_int4_linear(x, ldx, dtype, w, s, gs, T, C, R, bias, act, res, ldres, y, z, None, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(x=None), b"null"), (dict(w=None), b"null"), (dict(s=None), b"null"), (dict(y=None), b"null"),
    (dict(dtype=F32), b"bf16 or fp16"), (dict(dtype=7), b"bf16 or fp16"), (dict(C=60), b"multiple of 8"),
    (dict(C=0), b"bad sizes"), (dict(R=0), b"bad sizes"), (dict(T=-1), b"bad sizes"), (dict(R=1 << 25), b"bad sizes"),
    (dict(gs=48), b"group size"), (dict(gs=0), b"group size"), (dict(act=4), b"activation"), (dict(act=-1), b"activation"),
    (dict(ldx=56), b"row stride"), (dict(ldx=68), b"row stride"), (dict(x=FAKE + 2), b"aligned"),
    (dict(res=FAKE, ldres=15), b"residual"), (dict(y=FAKE + 8), b"aligned"), (dict(z=FAKE + 2), b"aligned")])
def test_linear_refuses(lib, kw, msg):
    assert _linear(lib, **kw) == 1
    assert msg in lib.forge_last_error()


def test_no_tokens_is_no_work(lib):
    assert _linear(lib, T=0, x=None, y=None) == 0
    assert lib.forge_int4_gated(None, 64, BF16, None, None, None, None, 32, 0, 64, 16, 2, None, None, None, None, None) == 0
    assert lib.forge_rmsnorm(None, 8, None, 0, None, BF16, BF16, 0, 8, 1e-6, None, None, None, None) == 0


def test_gated_refuses(lib):
    def call(x=FAKE, gw=FAKE, gs_=FAKE, uw=FAKE, us=FAKE, h=FAKE, g=None, u=None, gs=64, act=2):
        return lib.forge_int4_gated(x, 64, F16, gw, gs_, uw, us, gs, 2, 64, 16, act, h, g, u, None, None)
    for kw in (dict(x=None), dict(gw=None), dict(gs_=None), dict(uw=None), dict(us=None), dict(h=None), dict(g=FAKE),
               dict(u=FAKE), dict(gs=16), dict(act=9), dict(g=FAKE + 4, u=FAKE)):
        assert call(**kw) == 1, kw


def test_backward_refuses(lib):
    def lin(dy=FAKE, lddy=16, w=FAKE, s=FAKE, z=FAKE, act=2, dx=FAKE, db=None, ws=FAKE):
        return lib.forge_int4_linear_backward(dy, lddy, BF16, w, s, 32, 2, 64, 16, z, act, dx, db, ws, None, None)
    for kw in (dict(dy=None), dict(lddy=15), dict(w=None), dict(s=None), dict(z=None), dict(dx=None), dict(ws=None),
               dict(ws=FAKE + 16), dict(dx=FAKE + 2)):
        assert lin(**kw) == 1, kw

    def gat(dh=FAKE, lddh=16, g=FAKE, u=FAKE, w=FAKE, dx=FAKE, ws=FAKE):
        return lib.forge_int4_gated_backward(dh, lddh, BF16, g, u, w, FAKE, FAKE, FAKE, 32, 2, 64, 16, 2, dx, ws, None, None)
    for kw in (dict(dh=None), dict(lddh=8), dict(g=None), dict(u=None), dict(w=None), dict(dx=None), dict(ws=None),
               dict(ws=FAKE + 16)):
        assert gat(**kw) == 1, kw


def test_norm_refuses(lib):
    def fwd(x=FAKE, ldx=64, res=None, ldres=0, w=FAKE, wd=BF16, d=BF16, T=2, C=64, y=FAKE, s=None, r=None):
        return lib.forge_rmsnorm(x, ldx, res, ldres, w, wd, d, T, C, 1e-6, y, s, r, None)
    for kw in (dict(x=None), dict(w=None), dict(y=None), dict(ldx=63), dict(res=FAKE, ldres=64), dict(r=FAKE),
               dict(res=FAKE, r=FAKE, ldres=1), dict(wd=F16), dict(d=5), dict(C=0), dict(T=-1)):
        assert fwd(**kw) == 1, kw

    def bwd(dy=FAKE, lddy=64, x=FAKE, ldx=64, w=FAKE, wd=BF16, dres=None, lddres=0, dx=FAKE, dw=FAKE, ws=FAKE, C=64):
        return lib.forge_rmsnorm_backward(dy, lddy, x, ldx, w, wd, BF16, dres, lddres, 2, C, 1e-6, dx, dw, ws, None)
    for kw in (dict(dy=None), dict(x=None), dict(w=None), dict(dx=None), dict(dw=None), dict(ws=None), dict(ws=FAKE + 4),
               dict(lddy=1), dict(ldx=1), dict(dres=FAKE, lddres=1), dict(wd=F16), dict(C=-1)):
        assert bwd(**kw) == 1, kw


def test_workspace_sizes_cover_every_array(lib):
    for T, C, R, gs, mats in ((1, 8, 1, 32, 1), (5, 776, 1001, 32, 2), (4096, 7168, 2048, 128, 2), (0, 64, 64, 64, 1)):
        n = lib.forge_int4_backward_workspace_bytes(T, C, R, gs, mats)
        K = -(-mats * R // 64) * 64
        assert n >= T * K * 2 + T * 4 + mats * R * (-(-C // gs)) * 4 + mats * R * 4
    assert lib.forge_int4_backward_workspace_bytes(1, 8, 8, 0, 1) == 0
    for T, C in ((1, 1), (16, 7168), (5003, 2048), (100000, 64), (3, 20001)):
        assert lib.forge_rmsnorm_backward_workspace_bytes(T, C) >= 4 * C


def test_python_wrappers_refuse_cpu_tensors():
    from forge import ops
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w, s = torch.zeros(16, 8, dtype=torch.int32), torch.ones(16, 2)
    for call in (lambda: ops.rmsnorm(x, x[0]), lambda: ops.rmsnorm_backward(x, x, x[0]),
                 lambda: ops.int4_linear(x, w, s, 32), lambda: ops.int4_gated(x, w, s, w, s, 32),
                 lambda: ops.int4_linear_backward(x[:, :16], w, s, 32),
                 lambda: ops.int4_gated_backward(x[:, :16], x, x, w, s, w, s, 32)):
        with pytest.raises(RuntimeError):
            call()


def test_feed_forward_block_checks_its_matrices():
    from forge.inference import Int4FeedForward
    gate = (torch.zeros(16, 8, dtype=torch.int32), torch.ones(16, 2))
    down = (torch.zeros(64, 2, dtype=torch.int32), torch.ones(64, 1))
    up = tuple(t.clone() for t in gate)
    blk = Int4FeedForward(gate, up, down, group_size=32)
    assert sorted(n for n, _ in blk.named_buffers()) == ["down_packed", "down_scales", "gate_packed", "gate_scales",
                                                         "up_packed", "up_scales"]
    third = up[1] / 3
    blk.up_scales.copy_(third)
    blk = blk.to(torch.bfloat16).half()              # the scales stay as they are
    assert blk.up_scales.dtype == torch.float32 and torch.equal(blk.up_scales, third)
    with pytest.raises(RuntimeError):
        Int4FeedForward(gate, gate, gate, group_size=32)
    with pytest.raises(RuntimeError):
        Int4FeedForward(gate, down, down, group_size=32)
    with pytest.raises(RuntimeError):
        blk(torch.zeros(1, 64, dtype=torch.bfloat16), residual=torch.zeros(1, 64, dtype=torch.bfloat16))
