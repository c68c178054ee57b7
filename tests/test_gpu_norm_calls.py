"""The norm called from several threads, and rows of every length by the form that reads them once.

Tolerances, derived before the first run: half a step of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24) and, for the fp32
statistics, at most 64 additions in a thread and ten joins, 2^-24 each, half of that in the root."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
EPS = 1e-6
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
STAT = 48 * 2.0 ** -24


def ops():
    from forge import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def test_threads_whose_rows_need_different_shared_memory():
    """One kernel, launched by four threads at once with and without a residual and with rows of different lengths, through
    the C entry point: its argument conversion leaves the threads more time side by side inside the library."""
    from forge import _abi
    lib = _abi.load_library()
    g = gen(1)
    cases = []
    for C in (8192, 6144, 8192, 4096):
        x, r = (torch.randn(1, C, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
        w = torch.ones(C, device=DEV, dtype=torch.bfloat16)
        y, h = torch.empty_like(x), torch.empty_like(x)
        res = len(cases) % 2 == 0
        cases.append((x, w, r if res else None, y))
        cases[-1] += ((x.data_ptr(), C, r.data_ptr() if res else None, C, w.data_ptr(), _abi.BF16, _abi.BF16, 1, C, EPS,
                       y.data_ptr(), None, h.data_ptr() if res else None), h)
    bad = []
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()

    def work(i):
        fn, args, st = lib.forge_rmsnorm, cases[i][4], streams[i].cuda_stream
        for _ in range(5000):
            rc = fn(*args, st)
            if rc != 0:
                bad.append((i, rc, lib.forge_last_error()))
                return
    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    torch.cuda.synchronize()
    assert not bad, bad
    for x, w, r, y, _, h in cases:
        got = ops().rmsnorm(x, w, EPS, residual=r)
        assert torch.equal(got if r is None else got[0], y) and (r is None or torch.equal(got[1], h))


@pytest.mark.parametrize("T,C", [(3, 8200), (400, 8200), (301, 12288), (2, 16376), (333, 16384), (310, 4104), (299, 8192)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
def test_long_rows(T, C, dt, residual):
    """Two vectors of a row per thread, several rows per CTA, against float64; the 8-bit form against the formula at its own
    scales; a row of NaN and a row of zeros spoil nothing beside them."""
    g = gen(T + C)
    x, w = torch.randn(T, C, generator=g, device=DEV).to(dt), torch.randn(C, generator=g, device=DEV).to(dt)
    res = torch.randn(T, C, generator=g, device=DEV).to(dt) if residual else None
    x[T // 2, 3] = float("nan")
    x[0] = 0
    if residual:
        res[0] = 0
    h = x.double() + (res.double() if residual else 0)
    want = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * w.double()
    good = torch.arange(T, device=DEV) != T // 2
    got = ops().rmsnorm(x, w, EPS, residual=res)
    y, r = got if residual else (got, None)
    # with a residual h is an fp32 sum: 2^-24 of it more
    tol = (HALF[dt] + STAT + 2.0 ** -23) * want.abs() + 1e-7 * (dt == torch.float16)
    assert bool(((y.double() - want).abs() <= tol)[good].all()) and bool(y[T // 2].isnan().all())
    assert not bool(y[0].any())
    if residual:
        assert bool(((r.double() - h).abs() <= (HALF[dt] + 2.0 ** -23) * h.abs() + 1e-7 * (dt == torch.float16))[good].all())
    if dt == torch.float32:
        return
    q, s, *rest = ops().rmsnorm(x, w, EPS, residual=res, quant_group=128)
    assert not residual or torch.equal(rest[0][good], r[good])
    step = s.double().repeat_interleave(128, 1)[:, :C]
    groups = torch.nn.functional.pad(want, (0, -C % 128)).view(T, -1, 128).abs().amax(2).clamp_min(1e-12) / 448
    assert bool(((s.double() - groups).abs() <= 2.0 ** -18 * groups)[good].all())
    # half a step of e4m3 (2^-4 relative, 2^-10 of the scale among its subnormals) and the fp32 roundings before it
    assert bool(((q.double() * step - want).abs() <= (2.0 ** -4 + 2.0 ** -17) * want.abs() + 2.0 ** -10 * step)[good].all())


@pytest.mark.parametrize("T,C", [(300, 64), (300, 384), (200, 1000), (40, 4096), (40, 4100), (20, 9000), (20, 9001)])
def test_eight_bits_are_the_rounded_quotient(T, C):
    """scale = max |y| / 448 bit for bit, and q = e4m3(y / scale) from the y that the same rows give in fp32.  The kernel
    multiplies by the scale's rounded reciprocal: the product is within 3 2^-24 of the quotient, so rounding keeps it between
    the codes of the quotient times 1 -+ 2^-22.  (The oracle divides in float64, since torch divides an fp32 tensor by a
    number as a product with the rounded inverse.)"""
    g = gen(C)
    x, w = torch.randn(T, C, generator=g, device=DEV), torch.randn(C, generator=g, device=DEV)
    y = ops().rmsnorm(x, w, EPS)
    q, s = ops().rmsnorm(x, w, EPS, quant_group=128)
    groups = torch.nn.functional.pad(y, (0, -C % 128)).view(T, -1, 128)
    want_s = (groups.abs().amax(2).clamp_min(1e-12).double() / 448).float()
    assert torch.equal(s, want_s)
    quot = groups.double() / want_s.double().unsqueeze(2)
    code = lambda v: v.float().to(torch.float8_e4m3fn).float().view(T, -1)[:, :C]
    lo, hi = code(quot * (1 - 2.0 ** -22)), code(quot * (1 + 2.0 ** -22))
    got = q.float()
    assert bool(((got >= torch.minimum(lo, hi)) & (got <= torch.maximum(lo, hi))).all())
    assert float((lo != hi).float().mean()) < 1e-4


@pytest.mark.parametrize("T,C", [(6000, 264), (3001, 384), (5000, 512), (900, 8192), (700, 8200), (65, 16384)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_backward_of_many_rows(T, C, dt):
    """More rows than warps or CTAs walk at once, norm-wise against float64: one rounding of dx and of dweight (h / sqrt(3) of
    the norm and a tenth), fp32 sums over a row (2^-18) and over T rows (2^-24 each at most, of magnitudes that are
    sqrt(T) times the sum's)."""
    g = gen(T)
    x, dy, dres = (torch.randn(T, C, generator=g, device=DEV).to(dt) for _ in range(3))
    w = (1 + 0.3 * torch.randn(C, generator=g, device=DEV)).to(dt)
    X, t = x.double(), dy.double() * w.double()
    rstd = 1 / torch.sqrt(X.square().mean(1, keepdim=True) + EPS)
    n = X * rstd
    dx64 = rstd * (t - n * (t * n).mean(1, keepdim=True))
    dw64 = (dy.double() * n).sum(0)
    one = 1.1 * HALF[dt] / 3 ** 0.5
    off = lambda a, b: float((a.double() - b).norm() / b.norm())
    dx, dw = ops().rmsnorm_backward(dy, x, w, EPS)
    assert off(dx, dx64) <= one + 2.0 ** -18 and off(dw, dw64) <= one + T ** 0.5 * 2.0 ** -21
    dx, dw2 = ops().rmsnorm_backward(dy, x, w, EPS, dresidual=dres)
    assert off(dx, dx64 + dres.double()) <= one + 2.0 ** -18 and torch.equal(dw, dw2)
