"""The norm, the int4 products and the feed-forward block made of them, against the formulas in float64.

Tolerances, derived before the first run.  Output in type t: half a step, eps_t / 2 relative to the value (bf16 2^-8,
fp16 2^-11).  fp32 sums: a sum of n products is off by at most n 2^-23 of the sum of magnitudes when every addition
truncates; the kernels sum at most 256 products before adding the partial result, rounded, to a running sum over the
groups, so (256 2^-23 + G 2^-24) of |x| |W|^T covers every variant.  dz enters its product as fp16 (2^-11), so does the
weight (2^-11, for bf16 gradients from a scale rounded to fp16 too, 2^-11 more): 2^-10, or 3 2^-11, of |dz| |W| more for dx.  Activations: |act'| <= 1.13, a few fp32 roundings."""
import math

import pytest
import torch

from forge import _abi

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
EPS = 1e-6


def ops():
    from forge import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def weight(R, C, gs, g, spread=1.0):
    codes = torch.randint(0, 16, (R, C), generator=g, device=DEV, dtype=torch.int32)
    G = -(-C // gs)
    scales = torch.exp(spread * torch.randn(R, G, generator=g, device=DEV)) / (5 * math.sqrt(C))
    packed = torch.zeros(R, C // 8, dtype=torch.int32, device=DEV)
    for i in range(8):
        packed |= codes[:, i::8] << (4 * i)
    W = (codes.double() - 8) * scales.double().repeat_interleave(gs, 1)[:, :C]
    return packed, scales, W


def sum_tol(x, W, G):
    return (256 * 2.0 ** -23 + G * 2.0 ** -24) * (x.abs() @ W.abs().T)


def act64(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z


def dact64(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def close(got, want, tol, what=""):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                                 f"{float(got[bad][0])} for {float(want[bad][0])}, tolerance {float(tol.expand_as(want)[bad][0])}")


# ---- norm --------------------------------------------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (1, 8), (3, 129), (5, 256), (9, 264), (2, 512), (7, 1000), (4, 1024), (3, 1032), (3, 2048), (2, 2056),
               (2, 4096), (3, 7168), (1, 8192), (2, 8200), (1, 16384), (1, 16392), (2, 20001)]


def norm64(h, w):
    return h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * w


@pytest.mark.parametrize("T,C", NORM_SHAPES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_norm(T, C, dt):
    g = gen(C)
    x, res = torch.randn(T, C, generator=g, device=DEV).to(dt), (3 * torch.randn(T, C, generator=g, device=DEV)).to(dt)
    for wt in {dt, torch.float32}:
        w = (1 + 0.3 * torch.randn(C, generator=g, device=DEV)).to(wt)
        want = norm64(x.double(), w.double())
        # fp32 statistics: at most 64 sequential additions in a thread and ten joins, each 2^-24, half of that in the root
        rel = HALF[dt] + 48 * 2.0 ** -24
        close(ops().rmsnorm(x, w, EPS), want, rel * want.abs() + 1e-7 * (dt == torch.float16), "y")
        h = x.double() + res.double()
        y, r = ops().rmsnorm(x, w, EPS, residual=res)
        want = norm64(h, w.double())
        close(y, want, (rel + 2.0 ** -23) * want.abs() + 2.0 ** -24 * h.abs().max() * w.double().abs().max()
              / h.square().mean(1, keepdim=True).sqrt() + 1e-7 * (dt == torch.float16), "y")
        close(r, h, (HALF[dt] + 2.0 ** -23) * h.abs() + 2.0 ** -24 * h.abs().max() + 1e-7 * (dt == torch.float16), "h")


@pytest.mark.parametrize("T,C", NORM_SHAPES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_norm_eight_bits(T, C, dt):
    g = gen(C + 1)
    x, w = torch.randn(T, C, generator=g, device=DEV).to(dt), torch.randn(C, generator=g, device=DEV).to(dt)
    x[0, : min(C, 128)] = 0          # a group of zeros
    q, s = ops().rmsnorm(x, w, EPS, quant_group=128)
    assert q.dtype == torch.float8_e4m3fn and s.shape == (T, -(-C // 128))
    y = norm64(x.double(), w.double())
    pad = torch.nn.functional.pad(y, (0, -C % 128)).view(T, -1, 128)
    want_s = pad.abs().amax(2).clamp_min(1e-12) / 448
    close(s, want_s, 2.0 ** -18 * want_s, "scales")
    step = s.double().repeat_interleave(128, 1)[:, :C]
    # half a step of e4m3 (2^-4 relative, 2^-10 of the scale among its subnormals), and the fp32 roundings before it
    close(q.double() * step, y, 2.0 ** -4 * (1 + 2.0 ** -16) * y.abs() + 2.0 ** -10 * step + 2.0 ** -18 * y.abs(), "q")
    if C % 128 == 0 or C < 128:      # the reader wants equal column tiles
        back = ops().fp8_block_dequant(q, s)
        close(back, q.double() * step, 2.0 ** -8 * (q.double() * step).abs() + 2.0 ** -24 * step, "dequantised")
    y2, s2, h = ops().rmsnorm(x, w, EPS, residual=torch.zeros_like(x), quant_group=128)
    assert torch.equal(y2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s) and torch.equal(h, x)


@pytest.mark.parametrize("T,C", NORM_SHAPES + [(0, 64), (700, 320), (1200, 2048), (333, 775)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_backward(T, C, dt):
    g = gen(C + 2)
    x, dy, dr = (torch.randn(T, C, generator=g, device=DEV).to(dt) for _ in range(3))
    w = (1 + 0.3 * torch.randn(C, generator=g, device=DEV)).to(dt)
    X, DY, Wd = x.double(), dy.double(), w.double()
    rstd = 1 / torch.sqrt(X.square().mean(1, keepdim=True) + EPS)
    n, t = X * rstd, DY * Wd
    dx = rstd * (t - n * (t * n).mean(1, keepdim=True))
    mag = rstd * (t.abs() + n.abs() * (t * n).abs().mean(1, keepdim=True))
    tiny = 1e-7 * (dt == torch.float16)
    got, dw = ops().rmsnorm_backward(dy, x, w, EPS)
    close(got, dx, HALF[dt] * dx.abs() + 128 * 2.0 ** -24 * mag + tiny, "dx")
    want = (DY * n).sum(0)
    close(dw, want, HALF[dt] * want.abs() + (64 + max(T, 1) / 4) * 2.0 ** -24 * (DY * n).abs().sum(0) + tiny, "dweight")
    assert dw.dtype == w.dtype and (T > 0 or not bool(dw.any()))
    got, dw2 = ops().rmsnorm_backward(dy, x, w, EPS, dresidual=dr)
    dx = dx + dr.double()
    close(got, dx, HALF[dt] * dx.abs() + 128 * 2.0 ** -24 * (mag + dr.double().abs()) + tiny, "dx + dresidual")
    assert torch.equal(dw, dw2)


def test_norm_backward_against_differences():
    g = gen(5)
    T, C = 3, 520
    x, dy, w = (torch.randn(*s, generator=g, device=DEV) for s in ((T, C), (T, C), (C,)))
    dx, dw = ops().rmsnorm_backward(dy, x, w, EPS)
    X, D, Wd, h = x.double(), dy.double(), w.double(), 1e-5
    for k in range(4):
        v, vw = torch.randn(T, C, generator=g, device=DEV).double(), torch.randn(C, generator=g, device=DEV).double()
        num = ((norm64(X + h * v, Wd) - norm64(X - h * v, Wd)) * D).sum() / (2 * h)
        assert abs(float(num - (dx.double() * v).sum())) <= 1e-4 * float((dx.double() * v).abs().sum())
        num = ((norm64(X, Wd + h * vw) - norm64(X, Wd - h * vw)) * D).sum() / (2 * h)
        assert abs(float(num - (dw.double() * vw).sum())) <= 1e-4 * float((dw.double() * vw).abs().sum())


@pytest.mark.parametrize("C", [320, 1000, 2048])
def test_norm_strided_rows_and_bad_rows(C):
    g = gen(9)
    base = torch.randn(6, 2 * C + 3, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randn(C, generator=g, device=DEV).to(torch.bfloat16)
    for view in (base[:, :C], base[:, 1:1 + C], base[:, C + 3:], base[::2, 8:8 + C], base.t()[:C, :].t(), base[:1].expand(6, -1)[:, :C]):
        want = norm64(view.double(), w.double())
        close(ops().rmsnorm(view, w, EPS), want, (2.0 ** -8 + 2.0 ** -18) * want.abs())
        dx, dw = ops().rmsnorm_backward(view, view, w, EPS, dresidual=view)
        dx2, dw2 = ops().rmsnorm_backward(*(view.clone(memory_format=torch.contiguous_format),) * 2, w, EPS,
                                          dresidual=view.clone(memory_format=torch.contiguous_format))
        close(dx, dx2.double(), 2.0 ** -7 * dx2.double().abs() + 1e-5)
        close(dw, dw2.double(), 2.0 ** -7 * dw2.double().abs() + 1e-3)
    x = base[:, :C].contiguous()
    clean = ops().rmsnorm(x, w, EPS)
    x[1, 3], x[3, 5], x[4] = float("nan"), float("inf"), 0
    y, (q, s) = ops().rmsnorm(x, w, EPS), ops().rmsnorm(x, w, EPS, quant_group=128)
    assert bool(y[1].isnan().all()) and bool(s[1].isnan().all()) and bool(y[3, 5].isnan()) and not bool(y[4].any())
    assert not bool(q[4].float().any()) and torch.equal(s[4], torch.full_like(s[4], 1e-12) / 448)
    for r in (0, 2, 5):
        assert torch.equal(y[r], clean[r])


# ---- products ----------------------------------------------------------------------------------------------------------
TOKENS = [1, 2, 3, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 256, 300]
SHAPES = [(8, 1), (8, 16), (16, 5), (40, 17), (64, 64), (96, 33), (128, 128), (136, 129), (256, 255), (264, 300), (520, 96),
          (776, 1001), (1032, 260), (2048, 40)]
COMBOS = [(T, *SHAPES[(i + j) % len(SHAPES)], (32, 64, 128)[(i + j) % 3], (torch.bfloat16, torch.float16)[(i * 3 + j) % 2],
           ("none", "relu", "silu", "gelu")[(i + 2 * j) % 4]) for i, T in enumerate(TOKENS) for j in (0, 3, 7, 12)]


def check_linear(T, C, R, gs, dt, act, g, x=None, bias=True, residual=True):
    packed, scales, W = weight(R, C, gs, g)
    if x is None:
        x = torch.randn(T, C, generator=g, device=DEV).to(dt)
    b = torch.randn(R, generator=g, device=DEV).to(dt) if bias else None
    res = torch.randn(T, R, generator=g, device=DEV).to(dt) if residual else None
    y, z = ops().int4_linear(x, packed, scales, gs, bias=b, act=act, residual=res, want_preact=True)
    Z = x.double() @ W.T + (b.double() if bias else 0)
    tz = sum_tol(x.double(), W, scales.shape[1]) + 2.0 ** -23 * Z.abs()
    tiny = 2.0 ** -25 * (dt == torch.float16)
    close(z, Z, HALF[dt] * Z.abs() + tz + tiny, "preact")
    Y = act64(Z, act)
    ty = 1.13 * tz + 2.0 ** -20 * (Y.abs() + Z.abs() * 2.0 ** -2)
    if residual:
        Y = Y + res.double()
        ty = ty + 2.0 ** -23 * Y.abs()
    close(y, Y, HALF[dt] * Y.abs() + ty + tiny, "y")
    y2 = ops().int4_linear(x, packed, scales, gs, bias=b, act=act, residual=res)
    assert torch.equal(y, y2)
    return packed, scales, W, x


@pytest.mark.parametrize("T,C,R,gs,dt,act", COMBOS)
def test_linear(T, C, R, gs, dt, act):
    g = gen(T * 7919 + C)
    check_linear(T, C, R, gs, dt, act, g, bias=(T + R) % 2 == 0, residual=(T + C) % 3 != 0)


@pytest.mark.parametrize("T,C,R,gs,dt,act", COMBOS)
def test_gated(T, C, R, gs, dt, act):
    act = "silu" if act == "none" else act
    g = gen(T * 104729 + C)
    wg, sg, Wg = weight(R, C, gs, g)
    wu, su, Wu = weight(R, C, gs, g)
    x = torch.randn(T, C, generator=g, device=DEV).to(dt)
    h, gg, uu = ops().int4_gated(x, wg, sg, wu, su, gs, act=act, want_preact=True)
    X = x.double()
    Gt, Ut = X @ Wg.T, X @ Wu.T
    tg, tu = sum_tol(X, Wg, sg.shape[1]), sum_tol(X, Wu, su.shape[1])
    tiny = 2.0 ** -25 * (dt == torch.float16)
    close(gg, Gt, HALF[dt] * Gt.abs() + tg + tiny, "g")
    close(uu, Ut, HALF[dt] * Ut.abs() + tu + tiny, "u")
    A = act64(Gt, act)
    H = A * Ut
    th = (1.13 * tg + 2.0 ** -20 * (A.abs() + Gt.abs() / 4)) * Ut.abs() + A.abs() * tu + 2.0 ** -22 * H.abs()
    close(h, H, HALF[dt] * H.abs() + th + tiny, "h")
    assert torch.equal(h, ops().int4_gated(x, wg, sg, wu, su, gs, act=act))


def grad_tol(dz, W, dt, dx):
    return HALF[dt] * dx.abs() + ((3 if dt == torch.bfloat16 else 2) * 2.0 ** -11 + 2.0 ** -13) * (dz.abs() @ W.abs()) + 2.0 ** -25 * (dt == torch.float16)


@pytest.mark.parametrize("T,C,R,gs,dt,act", COMBOS)
def test_linear_backward(T, C, R, gs, dt, act):
    g = gen(T * 31 + R)
    packed, scales, W = weight(R, C, gs, g)
    z, dy = (torch.randn(T, R, generator=g, device=DEV).to(dt) for _ in range(2))
    dy[0] *= 2.0 ** -9           # rows of very different size
    dx, db = ops().int4_linear_backward(dy, packed, scales, gs, preact=z, act=act, want_dbias=True)
    dz = dy.double() * dact64(z.double(), act)
    want = dz @ W
    close(dx, want, grad_tol(dz, W, dt, want), "dx")
    want = dz.sum(0)
    # (below 2^-14 the step of fp16 stays 2^-24: half of it is 2^-25, whatever the value)
    close(db, want, HALF[dt] * want.abs() + (T + 64) * 2.0 ** -24 * dz.abs().sum(0) + 2.0 ** -20 * dy.double().abs().sum(0)
          + 2.0 ** -25 * (dt == torch.float16), "dbias")
    only, none = ops().int4_linear_backward(dy, packed, scales, gs, preact=z, act=act)
    assert none is None and torch.equal(only, dx)


@pytest.mark.parametrize("T,C,R,gs,dt,act", COMBOS)
def test_gated_backward(T, C, R, gs, dt, act):
    act = "silu" if act == "none" else act
    g = gen(T * 37 + R)
    wg, sg, Wg = weight(R, C, gs, g)
    wu, su, Wu = weight(R, C, gs, g)
    gg, uu, dh = (torch.randn(T, R, generator=g, device=DEV).to(dt) for _ in range(3))
    dx = ops().int4_gated_backward(dh, gg, uu, wg, sg, wu, su, gs, act=act)
    D, Gt, Ut = dh.double(), gg.double(), uu.double()
    dg, du = D * Ut * dact64(Gt, act), D * act64(Gt, act)
    want = dg @ Wg + du @ Wu
    close(dx, want, grad_tol(dg, Wg, dt, want) + grad_tol(du, Wu, dt, want * 0), "dx")


# enough tiles that two CTAs share each (more than 37 tiles of 256 rows x 256 tokens), with ragged edges in every direction
LARGE = [(1100, 264, 2501, 32, torch.bfloat16, "gelu"), (2049, 520, 1300, 64, torch.float16, "none"),
         (2600, 1032, 1025, 128, torch.bfloat16, "silu"), (257, 136, 5000, 128, torch.float16, "relu"),
         (3000, 8, 1000, 32, torch.bfloat16, "none")]


@pytest.mark.parametrize("T,C,R,gs,dt,act", LARGE)
def test_large_tiles(T, C, R, gs, dt, act):
    g = gen(T + C)
    packed, scales, W, x = check_linear(T, C, R, gs, dt, act, g)
    check_linear(T, C, R, gs, dt, "none", g, bias=False, residual=True)
    y = ops().int4_linear(x, packed, scales, gs)
    Z = x.double() @ W.T
    close(y, Z, HALF[dt] * Z.abs() + sum_tol(x.double(), W, scales.shape[1]) + 2.0 ** -25, "plain product")
    test_gated(T, C, R // 2 + 1, gs, dt, act)
    # the backward product has C on the side of the rows
    test_linear_backward(T, 8 * (R // 8), max(C, 33), gs, dt, act)
    test_gated_backward(T, 8 * (R // 8), max(C // 2 + 1, 33), gs, dt, act)


@pytest.mark.parametrize("T,C,R", [(5, 16384, 40), (20, 16384, 40), (40, 20000, 70), (130, 16384, 300), (700, 8200, 64)])
def test_long_sums_over_few_rows(T, C, R):
    """The K axis is shared by the warps or the CTAs of a cluster, unevenly."""
    test_linear(T, C, R, 128, torch.bfloat16, "none")
    test_gated(T, C, R, 64, torch.float16, "silu")
    test_linear_backward(T, 8 * R, C // 4, 32, torch.bfloat16, "gelu")


@pytest.mark.parametrize("T", [3, 20, 100])
def test_words_that_start_off_16_bytes(T):
    """Packed matrices that are views into one buffer: rows start on 4 or 8 bytes only."""
    g = gen(T + 1)
    C, R, gs = 256, 48, 128
    packed, scales, W = weight(R, C, gs, g)
    x = torch.randn(T, C, generator=g, device=DEV).half()
    want = ops().int4_linear(x, packed, scales, gs)
    want_g = ops().int4_gated(x, packed, scales, packed, scales, gs)
    dy = torch.randn(T, R, generator=g, device=DEV).half()
    want_d = ops().int4_linear_backward(dy, packed, scales, gs)[0]
    for off in (1, 2, 3, 4):
        buf = torch.zeros(packed.numel() + off, dtype=torch.int32, device=DEV)
        view = buf[off:].view(R, C // 8)
        view.copy_(packed)
        assert torch.equal(ops().int4_linear(x, view, scales, gs), want)
        assert torch.equal(ops().int4_gated(x, view, scales, packed, scales, gs), want_g)
        assert torch.equal(ops().int4_linear_backward(dy, view, scales, gs)[0], want_d)


def test_gated_backward_against_differences():
    g = gen(77)
    T, C, R, gs = 3, 128, 96, 32
    wg, sg, Wg = weight(R, C, gs, g)
    wu, su, Wu = weight(R, C, gs, g)
    x, dh = torch.randn(T, C, generator=g, device=DEV).half(), torch.randn(T, R, generator=g, device=DEV).half()
    _, gg, uu = ops().int4_gated(x, wg, sg, wu, su, gs, want_preact=True)
    dx = ops().int4_gated_backward(dh, gg, uu, wg, sg, wu, su, gs).double()
    X, D, e = x.double(), dh.double(), 1e-5
    f = lambda X: (act64(X @ Wg.T, "silu") * (X @ Wu.T) * D).sum()
    for _ in range(4):
        v = torch.randn(T, C, generator=g, device=DEV).double()
        # dx is off by fp16 roundings of g, u, dz, W and its own: 5 2^-11, in magnitudes
        mag = (D.abs() * 2 * ((X @ Wg.T).abs() + (X @ Wu.T).abs() + 1)) @ (Wg.abs() + Wu.abs())
        assert abs(float((f(X + e * v) - f(X - e * v)) / (2 * e) - (dx * v).sum())) <= 5 * 2.0 ** -11 * float((mag * v.abs()).sum())


@pytest.mark.parametrize("T", [1, 5, 40, 130])
def test_strides_extremes_and_bad_rows(T):
    g = gen(T)
    C, R, gs = 264, 136, 64
    packed, scales, W = weight(R, C, gs, g)
    base = torch.randn(T, 2 * C + 16, generator=g, device=DEV).to(torch.bfloat16)
    resb = torch.randn(T, R + 3, generator=g, device=DEV).to(torch.bfloat16)
    for x in (base[:, :C], base[:, 8:8 + C], base[:, 1:1 + C], base[:, C + 16:], base[:1].expand(T, -1)[:, :C]):
        dense = x.clone(memory_format=torch.contiguous_format)
        res = resb[:, 3:]
        got = ops().int4_linear(x, packed, scales, gs, residual=res)
        assert torch.equal(got, ops().int4_linear(dense, packed, scales, gs, residual=res.contiguous()))
    dyb = torch.randn(T, R + 5, generator=g, device=DEV).to(torch.bfloat16)
    assert torch.equal(ops().int4_linear_backward(dyb[:, 5:], packed, scales, gs)[0],
                       ops().int4_linear_backward(dyb[:, 5:].contiguous(), packed, scales, gs)[0])
    # extreme codes and scales: all -8, all 7, zero and negative scales, scales far apart in a row
    x = torch.randn(T, C, generator=g, device=DEV).to(torch.bfloat16)
    for word in (0, 0x77777777, -1, -0x77777778):      # codes 0, 7, 15, 8
        pk = torch.full_like(packed, word)
        sc = scales.clone()
        sc[0], sc[1], sc[2, ::2], sc[3] = 0, -sc[1], sc[2, ::2] * 1e-4, 1e-30
        Wx = float((word & 15) - 8) * sc.double().repeat_interleave(gs, 1)[:, :C]
        y = ops().int4_linear(x, pk, sc, gs)
        want = x.double() @ Wx.T
        close(y, want, 2.0 ** -8 * want.abs() + sum_tol(x.double(), Wx, 5), "extreme")
        dz = torch.randn(T, R, generator=g, device=DEV).to(torch.bfloat16)
        want = dz.double() @ Wx
        close(ops().int4_linear_backward(dz, pk, sc, gs)[0], want, grad_tol(dz.double(), Wx, torch.bfloat16, want)
              + 2.0 ** -24 * (dz.double().abs() @ Wx.abs().amax(1, keepdim=True).expand(R, C)), "extreme dx")
    # a bad token spoils its own row only; a row of zeros gives the bias
    clean = ops().int4_linear(x, packed, scales, gs)
    bad = x.clone()
    bad[T // 2, 5] = float("nan")
    y = ops().int4_linear(bad, packed, scales, gs)
    assert bool(y[T // 2].isnan().all())
    keep = [i for i in range(T) if i != T // 2]
    assert torch.equal(y[keep], clean[keep])
    dz = torch.randn(T, R, generator=g, device=DEV).to(torch.bfloat16)
    cleand = ops().int4_linear_backward(dz, packed, scales, gs)[0]
    dz[T // 2, 3] = float("inf")
    d = ops().int4_linear_backward(dz, packed, scales, gs)[0]
    assert not bool(d[T // 2].isfinite().any()) and torch.equal(d[keep], cleand[keep])
    dz[T // 2] = 0
    d = ops().int4_linear_backward(dz, packed, scales, gs)[0]
    assert not bool(d[T // 2].any()) and torch.equal(d[keep], cleand[keep])


def test_refusals():
    o, g = ops(), gen(0)
    packed, scales, _ = weight(16, 64, 32, g)
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    cases = [lambda: o.int4_linear(x[:, :56], packed, scales, 32), lambda: o.int4_linear(x.float(), packed, scales, 32),
             lambda: o.int4_linear(x, packed, scales, 64), lambda: o.int4_linear(x, packed, scales, 16),
             lambda: o.int4_linear(x, packed.t(), scales, 32), lambda: o.int4_linear(x, packed.long(), scales, 32),
             lambda: o.int4_linear(x, packed, scales, 32, act="tanh"), lambda: o.int4_linear(x, packed.cpu(), scales, 32),
             lambda: o.int4_linear(x, packed, scales, 32, bias=x[0, :15]),
             lambda: o.int4_linear(x, packed, scales, 32, bias=x[0, :16].float()),
             lambda: o.int4_linear(x, packed, scales, 32, residual=x),
             lambda: o.int4_linear(x[0], packed, scales, 32),
             lambda: o.int4_linear_backward(x[:, :16], packed, scales, 32, act="silu"),
             lambda: o.int4_linear_backward(x[:, :16], packed, scales, 32, want_dx=False),
             lambda: o.int4_linear_backward(x, packed, scales, 32),
             lambda: o.int4_gated(x, packed, scales, packed[:8], scales[:8], 32),
             lambda: o.int4_gated_backward(x[:, :16], x[:, :16], x, packed, scales, packed, scales, 32),
             lambda: o.rmsnorm(x, x[0, :63]), lambda: o.rmsnorm(x, x[0].half()), lambda: o.rmsnorm(x, x[0], quant_group=64),
             lambda: o.rmsnorm(x, x[0], residual=x[:1]), lambda: o.rmsnorm(x, x[0], residual=x.half()),
             lambda: o.rmsnorm(x[0], x[0]), lambda: o.rmsnorm(x.double(), x[0].double()),
             lambda: o.rmsnorm_backward(x, x[:1], x[0]), lambda: o.rmsnorm_backward(x.half(), x, x[0])]
    for i, c in enumerate(cases):
        with pytest.raises(RuntimeError):
            c()
            pytest.fail(f"case {i} was not refused", pytrace=False)
    # no tokens
    e = x[:0]
    assert o.int4_linear(e, packed, scales, 32).shape == (0, 16) and o.rmsnorm(e, x[0]).shape == (0, 64)
    assert o.int4_gated(e, packed, scales, packed, scales, 32).shape == (0, 16)
    dx, db = o.int4_linear_backward(e[:, :16], packed, scales, 32, want_dbias=True)
    assert dx.shape == (0, 64) and not bool(db.any())
    assert o.int4_gated_backward(*(e[:, :16],) * 3, packed, scales, packed, scales, 32).shape == (0, 64)


def block_parts(T, H, I, gs, dt, seed):
    g = gen(seed)
    parts = [weight(*s, gs, g, 0.3) for s in ((I, H), (I, H), (H, I))]
    x, res = (torch.randn(T, H, generator=g, device=DEV).to(dt) for _ in range(2))
    w = (1 + 0.2 * torch.randn(H, generator=g, device=DEV)).to(dt)
    return parts, x, res, w


def block64(parts, h, w):
    (_, _, Wg), (_, _, Wu), (_, _, Wd) = parts
    y = norm64(h, w)
    return (act64(y @ Wg.T, "silu") * (y @ Wu.T)) @ Wd.T + h


@pytest.mark.parametrize("T", [1, 20, 150])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_feed_forward_block(T, dt):
    """norm -> gated product -> product with the residual, forward and backward through autograd."""
    from forge.inference import Int4FeedForward
    H, I, gs = 256, 192, 64
    parts, x, res, w = block_parts(T, H, I, gs, dt, T)
    blk = Int4FeedForward(*[p[:2] for p in parts], group_size=gs, norm_weight=w)
    with torch.no_grad():
        out = blk(x.view(T, 1, H), residual=res.view(T, 1, H)).view(T, H)
    h = x.double() + res.double()
    want = block64(parts, h, w.double())
    # five roundings to the type on the way (y, h, the gated product, the stream, the result), linear in magnitudes
    Y = norm64(h, w.double()).abs()
    inner = (Y @ parts[0][2].abs().T) * (Y @ parts[1][2].abs().T)
    close(out, want, 5 * HALF[dt] * (inner @ parts[2][2].abs().T + h.abs()) * 1.13, "block")
    xg, rg = x.clone().requires_grad_(), res.clone().requires_grad_()
    o2 = blk(xg, residual=rg)
    assert torch.equal(o2.detach(), out)
    dout = torch.randn(T, H, generator=gen(1), device=DEV).to(dt)
    o2.backward(dout)
    hd, wd = h.clone().requires_grad_(), w.double().requires_grad_()
    block64(parts, hd, wd).backward(dout.double())
    assert torch.equal(xg.grad, rg.grad)
    # relative to the size of the gradients: roundings of every stored intermediate, fewer than sixteen
    for got, ref in ((xg.grad, hd.grad), (blk.norm_weight.grad, wd.grad)):
        err = (got.double() - ref).norm() / ref.norm()
        assert float(err) <= 16 * HALF[dt] / math.sqrt(3), float(err)


def test_feed_forward_block_from_the_quantiser():
    """A shared expert of a layer that MoELayerQuantizer packed, run on its packed words."""
    from forge import moe, synth
    from forge.inference import Int4FeedForward
    o = ops()
    shape = synth.LayerShape("small", 4, 1, 256, 128, 512, 2)
    X = synth.student_t_activations(shape.tokens, shape.hidden, seed=3).cuda()
    ids = o.route_topk(synth.router_logits(shape, shape.tokens, seed=3).cuda(), 2, "softmax")
    Wg, Wu, Wd = synth.expert_weights(shape, range(5), seed=3)
    cfg = moe.MoEQuantConfig(bits=4, group_size=128, symmetric=True, rel_damp=0.01)
    out = moe.MoELayerQuantizer(cfg).quantize_experts(X, ids, Wg.cuda(), Wu.cuda(), Wd.cuda(), dense_tail=1)
    for i in (0, 4):
        blk = Int4FeedForward.from_quantized(out, i, group_size=128)
        y = blk(X[:70])
        D = [o.dequantize(out[f]["qweight"][i], out[f]["scales"][i].reshape(-1), out[f]["qzeros"][i].reshape(-1), 128).double()
             for f in ("gate", "up", "down")]
        x = X[:70].double()
        a = act64(x @ D[0].T, "silu") * (x @ D[1].T)
        want = a @ D[2].T
        mag = ((x.abs() @ D[0].abs().T) * (x.abs() @ D[1].abs().T)) @ D[2].abs().T
        close(y, want, 2.0 ** -8 * want.abs() + 2.0 ** -8 * (a.abs() @ D[2].abs().T) * 1.01 + 2.0 ** -14 * mag, "expert")


def test_other_streams_and_graphs():
    """Two captured graphs and an eager call, interleaved on different streams, give the eager results."""
    from forge.inference import Int4FeedForward
    parts, x, res, w = block_parts(40, 256, 192, 64, torch.bfloat16, 5)
    blk = Int4FeedForward(*[p[:2] for p in parts], group_size=64, norm_weight=w)
    dy = torch.randn(40, 192, generator=gen(8), device=DEV).to(torch.bfloat16)

    def step(x, res, dy):
        with torch.no_grad():
            out = blk(x, residual=res)
            dx, db = ops().int4_linear_backward(dy, *parts[0][:2], 64, preact=dy, act="gelu", want_dbias=True)
            return out, dx, db, *ops().rmsnorm_backward(dx, x, w, EPS), ops().int4_gated_backward(
                dy, dy, dy, *parts[0][:2], *parts[1][:2], 64)
    inputs = [(x, res, dy), (res, x, -dy)]
    want = [step(*i) for i in inputs]
    torch.cuda.synchronize()
    static = [tuple(torch.empty_like(t) for t in i) for i in inputs]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for s in static:
        with torch.cuda.stream(side):
            for t in s:
                t.zero_()
            step(*s)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs.append(step(*s))
        graphs.append(gr)
    for _ in range(3):
        for i in (0, 1):
            for t, v in zip(static[i], inputs[i]):
                t.copy_(v)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(3)]
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            eager = step(*inputs[0])
        torch.cuda.synchronize()
        for i in (0, 1):
            for a, b in zip(outs[i], want[i]):
                assert torch.equal(a, b)
        for a, b in zip(eager, want[0]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 9, 30, 70, 513])
def test_same_bits_twice(T):
    g = gen(T)
    C, R, gs = 2048, 264, 128
    packed, scales, _ = weight(R, C, gs, g)
    up, us, _ = weight(R, C, gs, g)
    x, dy = torch.randn(T, C, generator=g, device=DEV).half(), torch.randn(T, R, generator=g, device=DEV).half()
    def once():
        h, gg, uu = ops().int4_gated(x, packed, scales, up, us, gs, want_preact=True)
        dx, db = ops().int4_linear_backward(dy, packed, scales, gs, preact=gg, act="silu", want_dbias=True)
        return (ops().int4_linear(x, packed, scales, gs), h, gg, uu, dx, db,
                ops().int4_gated_backward(dy, gg, uu, packed, scales, up, us, gs), *ops().rmsnorm_backward(x, x, x[0], EPS))
    first = once()
    for _ in range(3):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)


def test_rows_past_two_to_the_31_elements():
    T, C, R = 310000, 64, 7168
    g = gen(3)
    packed, scales, W = weight(R, C, 32, g)
    x = torch.randn(T, C, generator=g, device=DEV).to(torch.bfloat16)
    assert T * R > 2 ** 31
    y = ops().int4_linear(x, packed, scales, 32)
    tail = torch.tensor([0, 1, T // 2, T - 130, T - 2, T - 1], device=DEV)
    want = x[tail].double() @ W.T
    close(y[tail], want, 2.0 ** -8 * want.abs() + sum_tol(x[tail].double(), W, 2), "tail")
    dx, _ = ops().int4_linear_backward(y, packed, scales, 32)
    dz = y[tail].double()
    want = dz @ W
    close(dx[tail], want, grad_tol(dz, W, torch.bfloat16, want), "dx tail")
    del dx
    w = torch.ones(R, dtype=torch.bfloat16, device=DEV)
    n = ops().rmsnorm(y, w, EPS)
    want = norm64(y[tail].double(), w.double())
    close(n[tail], want, (2.0 ** -8 + 2.0 ** -18) * want.abs(), "norm tail")
    assert _abi.query("forge_launch_count") > 0


def test_captured_training_step():
    """Forward and backward of the block in one graph, replayed with other inputs, against the eager step."""
    from forge.inference import Int4FeedForward
    parts, x, res, w = block_parts(300, 256, 192, 64, torch.bfloat16, 11)
    blk = Int4FeedForward(*[p[:2] for p in parts], group_size=64, norm_weight=w)
    dout = torch.randn(300, 256, generator=gen(2), device=DEV).to(torch.bfloat16)

    def step(a, b):
        out = blk(a, residual=b)
        return (out, *torch.autograd.grad(out, (a, b, blk.norm_weight), dout))
    sx, sr = torch.zeros_like(x).requires_grad_(), torch.zeros_like(res).requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(sx, sr)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(sx, sr)
    for a, b in ((x, res), (res, x)):
        with torch.no_grad():
            sx.copy_(a)
            sr.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = step(a.clone().requires_grad_(), b.clone().requires_grad_())
        for g1, g2 in zip(got, want):
            assert torch.equal(g1, g2)


def test_block_without_norm_and_without_tokens():
    from forge.inference import Int4FeedForward
    parts, x, res, w = block_parts(9, 128, 64, 32, torch.float16, 3)
    bare = Int4FeedForward(*[p[:2] for p in parts], group_size=32)
    X = x.double()
    a = act64(X @ parts[0][2].T, "silu") * (X @ parts[1][2].T)
    want = a @ parts[2][2].T
    mag = ((X.abs() @ parts[0][2].abs().T) * (X.abs() @ parts[1][2].abs().T)) @ parts[2][2].abs().T
    close(bare(x), want, 2.0 ** -11 * want.abs() + 2.0 ** -11 * 1.01 * (a.abs() @ parts[2][2].abs().T) + 2.0 ** -14 * mag + 2.0 ** -24, "bare")
    normed = Int4FeedForward(*[p[:2] for p in parts], group_size=32, norm_weight=w)
    for blk in (bare, normed):
        assert blk(x[:0]).shape == (0, 128)
        e = x[:0].clone().requires_grad_()
        blk(e).sum().backward()
        assert e.grad.shape == (0, 128)
    assert not bool(normed.norm_weight.grad.any())


def test_calls_from_two_threads():
    import threading
    g = gen(4)
    packed, scales, _ = weight(264, 2048, 128, g)
    xs = [torch.randn(T, 2048, generator=g, device=DEV).half() for T in (1, 12, 60, 400)]
    want = [ops().int4_linear(x, packed, scales, 128) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                k = (i + _) % len(xs)
                y = ops().int4_linear(xs[k], packed, scales, 128)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, want[k]):
                    bad.append(k)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_few_tokens_and_many_rows():
    """More row tiles than SMs for one token tile: a CTA walks several tiles alone."""
    test_linear(40, 264, 20001, 64, torch.bfloat16, "gelu")
    test_gated(50, 136, 10300, 128, torch.float16, "silu")
    test_linear_backward(33, 20008, 70, 32, torch.bfloat16, "relu")
    test_gated_backward(60, 20008, 33, 128, torch.float16, "gelu")
    test_linear(9, 64, 40003, 32, torch.float16, "none")


@pytest.mark.parametrize("T", [2, 30, 700])
def test_plain_gate_half_scales_and_status(T):
    """No activation on the gate; scales kept in 16 bits; the status word stays clear."""
    g = gen(T + 5)
    C, R, gs = 512, 1300, 128
    wg, sg, Wg = weight(R, C, gs, g)
    wu, su, Wu = weight(R, C, gs, g)
    sg, su = sg.half(), su.half()                       # as a checkpoint keeps them (weights off by 2^-11)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    x = torch.randn(T, C, generator=g, device=DEV).half()
    h, gg, uu = ops().int4_gated(x, wg, sg, wu, su, gs, act="none", want_preact=True, status=status)
    a, b = (ops().int4_linear(x, w, s.float(), gs, status=status) for w, s in ((wg, sg), (wu, su)))
    # the two entry points may share the K axis among different numbers of CTAs, so their fp32 sums differ by the sums'
    # tolerance each, and each is then rounded to fp16: half a step (2^-11) either side
    for p, q, W in ((gg, a, Wg), (uu, b, Wu)):
        close(p, q.double(), 2 * 2.0 ** -11 * 1.01 * q.double().abs() + 2 * 1.01 * sum_tol(x.double(), W, C // gs) + 2.0 ** -24)
    prod = gg.double() * uu.double()
    # g, u and h rounded: half a step relative (2^-11) each, but never less than 2^-25, half of fp16's smallest step, which g
    # passes on times u and u times g
    close(h, prod, 3.1 * 2.0 ** -11 * prod.abs() + 1.01 * 2.0 ** -25 * (1 + gg.double().abs() + uu.double().abs()))
    dh = torch.randn(T, R, generator=g, device=DEV).half()
    dx = ops().int4_gated_backward(dh, gg, uu, wg, sg, wu, su, gs, act="none", status=status)
    dz = (dh.double() * uu.double(), dh.double() * gg.double())
    d1, _ = ops().int4_linear_backward(dz[0].half(), wg, sg, gs, status=status)
    d2, _ = ops().int4_linear_backward(dz[1].half(), wu, su, gs, status=status)
    mag = sum(d.abs() @ ops().int4_packed_dequant(w ^ -0x77777778, s, (R, C), dtype=torch.float32).double().abs()
              for d, w, s in ((dz[0], wg, sg), (dz[1], wu, su)))
    close(dx, d1.double() + d2.double(), 5 * 2.0 ** -11 * mag + 2.0 ** -23)
    assert int(status) == 0
