"""How exact the backward products over packed int4 weights are: single sums with a known rounding, and norm-wise bounds.

Tolerances, derived before the first run.  A sum over k of terms with independent signs has a norm of the root of the sum of
the terms' squares, and so has the sum of their independent errors: a relative rounding of half a step h of every term
contributes h / sqrt(3) at most, norm-wise (an error spread evenly over the step).  For bf16 gradients dz and the weight are
rounded to fp16 (2^-11 each), and the result to its own type: sqrt((h_type^2 + 2 (2^-11)^2) / 3); for fp16 gradients dz and
the weight keep 22 bits, so the result's rounding is all: h_type / sqrt(3).  A tenth more covers the spread of the norms of a
few thousand entries and the fp32 sums."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ops():
    from forge import ops as o
    return o


def words(codes):
    packed = torch.zeros(codes.shape[0], codes.shape[1] // 8, dtype=torch.int32, device=DEV)
    for i in range(8):
        packed |= codes[:, i::8].to(torch.int32) << (4 * i)
    return packed


def norm_bound(dt):
    return 1.1 * math.sqrt((HALF[dt] ** 2 + (2 * 2.0 ** -22 if dt == torch.bfloat16 else 0)) / 3)


@pytest.mark.parametrize("T", [3, 70, 5000])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_both_halves_of_the_scale_reach_the_gradient(T, dt):
    """55 equal terms 7 s with s just below 1 + 2^-11.  Rounded to fp16, s is 1 and the sum is 385, a tie in bf16 that goes to
    384; 7 s rounded once is 7 + 2^-8, and the sum lies above the tie like the exact one, 385.17: 386."""
    R, C, gs = 55, 1024, 32
    s = 1 + 2.0 ** -11 - 2.0 ** -15
    packed = words(torch.full((R, C), 15, device=DEV))
    dy = torch.ones(T, R, device=DEV, dtype=dt)
    dx, _ = ops().int4_linear_backward(dy, packed, torch.full((R, C // gs), s, device=DEV), gs)
    want = R * 7 * s
    if dt == torch.bfloat16:
        assert bool((dx == 386).all()), dx.unique()
    else:
        assert bool(((dx.double() - want).abs() <= 2.0 ** -11 * want).all()), dx.unique()


def spread_scales(R, C, gs, g, ratio, where):
    """Scales of one size, but for the channels of the first group: in every row, in one block of 512 rows and in the rows
    behind it, or in every row by another power of two, they are `ratio` of the others."""
    s = torch.rand(R, C // gs, generator=g, device=DEV) + 0.5
    if where == "group":
        s[:, 0] *= ratio
    elif where == "block":
        s[512:, 0] *= ratio
        s[:512, 0] = 0                       # (their products would hide the small ones)
    else:
        s[:, 0] *= ratio
        s *= 2.0 ** torch.randint(-20, 21, (R, 1), generator=g, device=DEV)
    return s


@pytest.mark.parametrize("T", [3, 70, 1500])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("where", ["group", "block", "rows"])
@pytest.mark.parametrize("power", [-13, -16, -20, -26, -40])
def test_groups_of_small_scales_keep_their_gradient(T, dt, where, power):
    """The channels whose scales are far below those of the rest of their rows, judged by themselves.  fp16 gradients are
    scaled so that the small group's are of ordinary size (the others may overflow)."""
    R, C, gs = 1100, 2560, 128
    g = torch.Generator(device=DEV).manual_seed(1000 * T - power)
    lift = 2.0 ** -power if dt == torch.float16 else 1.0

    def matrix():
        codes = torch.randint(0, 16, (R, C), generator=g, device=DEV)
        s = spread_scales(R, C, gs, g, 2.0 ** power, where) * lift
        return words(codes), s, (codes[:, :gs].double() - 8) * s[:, :1].double()
    (p0, s0, W0), (p1, s1, W1) = matrix(), matrix()
    dy = torch.randn(T, R, generator=g, device=DEV).to(dt)
    if where == "rows":                      # terms of one size, as the powers of the rows meet those of the gradient
        dy = (dy.double() * 2.0 ** -14).to(dt)
    dx = ops().int4_linear_backward(dy, p0, s0, gs)[0][:, :gs].double()
    want = dy.double() @ W0
    assert float((dx - want).norm() / want.norm()) <= norm_bound(dt)
    gate, up = (torch.randn(T, R, generator=g, device=DEV).to(dt) for _ in range(2))
    dx = ops().int4_gated_backward(dy, gate, up, p0, s0, p1, s1, gs, act="relu")[:, :gs].double()
    on = (gate > 0).double()
    want = (dy.double() * up.double() * on) @ W0 + (dy.double() * gate.double() * on) @ W1
    assert float((dx - want).norm() / want.norm()) <= norm_bound(dt)


def test_scales_of_more_groups_than_fit_at_a_time():
    R, C, gs, T = 700, 40000, 32, 5
    g = torch.Generator(device=DEV).manual_seed(9)
    codes = torch.randint(0, 16, (R, C), generator=g, device=DEV)
    s = (torch.rand(R, C // gs, generator=g, device=DEV) + 0.5) * 2.0 ** (-30 * torch.rand(1, C // gs, generator=g, device=DEV))
    dy = torch.randn(T, R, generator=g, device=DEV).to(torch.bfloat16)
    dx = ops().int4_linear_backward(dy, words(codes), s, gs)[0].double().view(T, -1, gs)
    want = (dy.double() @ ((codes.double() - 8) * s.double().repeat_interleave(gs, 1))).view(T, -1, gs)
    # group by group: 160 entries each, so the ratio of two norms spreads by a tenth more
    assert float(((dx - want).norm(dim=(0, 2)) / want.norm(dim=(0, 2))).max()) <= 1.5 * norm_bound(torch.bfloat16)


@pytest.mark.parametrize("T", [1, 8, 13])
@pytest.mark.parametrize("C,R,gs", [(1024, 200, 32), (776, 3000, 32), (2048, 5001, 64), (4104, 2500, 128), (7168, 2400, 32)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_few_tokens_and_wide_matrices(T, C, R, gs, dt):
    """The few-token form with eight warps (few channels or many rows), norm-wise: the products are exact but for fp32 sums, so
    one rounding of the result is all, h / sqrt(3) of it and a tenth; the gated result passes act and a product in fp32."""
    g = torch.Generator(device=DEV).manual_seed(T * C + R)
    mats = []
    for _ in range(2):
        codes = torch.randint(0, 16, (R, C), generator=g, device=DEV)
        s = (torch.rand(R, -(-C // gs), generator=g, device=DEV) + 0.5) / (5 * math.sqrt(C))
        mats.append((words(codes), s, (codes.double() - 8) * s.double().repeat_interleave(gs, 1)[:, :C]))
    (p0, s0, W0), (p1, s1, W1) = mats
    x = torch.randn(T, C, generator=g, device=DEV).to(dt)
    X = x.double()
    bound = 1.1 * HALF[dt] / math.sqrt(3) + 2.0 ** -18
    y, want = ops().int4_linear(x, p0, s0, gs).double(), X @ W0.T
    assert float((y - want).norm() / want.norm()) <= bound
    h, u, v = ops().int4_gated(x, p0, s0, p1, s1, gs, want_preact=True)
    a = X @ W0.T
    want = a * torch.sigmoid(a) * (X @ W1.T)
    assert float((h.double() - want).norm() / want.norm()) <= bound
    assert torch.equal(u, ops().int4_linear(x, p0, s0, gs)) and float((v.double() - X @ W1.T).norm() / (X @ W1.T).norm()) <= bound


def matrix(R, C, gs, g):
    codes = torch.randint(0, 16, (R, C), generator=g, device=DEV)
    s = torch.exp(torch.randn(R, -(-C // gs), generator=g, device=DEV)) / (5 * math.sqrt(C))
    return words(codes), s, (codes.double() - 8) * s.double().repeat_interleave(gs, 1)[:, :C]


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("T,C,R,gs", [(24, 2048, 776, 128), (64, 776, 1001, 32), (130, 1032, 520, 64), (333, 776, 1001, 32),
                                      (1500, 2048, 2000, 128), (2100, 1000, 1800, 64)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_every_form_norm_wise(T, C, R, gs, dt):
    """Forward: one rounding of the result, the fp32 sums 2^-18 of its norm at most (256 truncating additions of terms whose
    signs are independent).  Backward: the bound above, with dz from the stored values."""
    g = torch.Generator(device=DEV).manual_seed(T + C)
    (p0, s0, W0), (p1, s1, W1) = matrix(R, C, gs, g), matrix(R, C, gs, g)
    x = torch.randn(T, C, generator=g, device=DEV).to(dt)
    fwd = 1.1 * HALF[dt] / math.sqrt(3) + 2.0 ** -17
    z = x.double() @ W0.T
    y, saved = ops().int4_linear(x, p0, s0, gs, act="gelu", want_preact=True)
    assert off(y, z * torch.special.ndtr(z)) <= fwd and off(saved, z) <= fwd
    assert off(ops().int4_linear(x, p0, s0, gs), z) <= fwd
    h, u, v = ops().int4_gated(x, p0, s0, p1, s1, gs, want_preact=True)
    assert off(h, z * torch.sigmoid(z) * (x.double() @ W1.T)) <= fwd and off(v, x.double() @ W1.T) <= fwd
    dy = torch.randn(T, R, generator=g, device=DEV).to(dt)
    Z = saved.double()
    dz = dy.double() * (torch.special.ndtr(Z) + Z * torch.exp(-Z * Z / 2) / math.sqrt(2 * math.pi))
    dx, db = ops().int4_linear_backward(dy, p0, s0, gs, preact=saved, act="gelu", want_dbias=True)
    assert off(dx, dz @ W0) <= norm_bound(dt) and off(db, dz.sum(0)) <= fwd
    U, V = u.double(), v.double()
    sig = torch.sigmoid(U)
    want = (dy.double() * V * sig * (1 + U * (1 - sig))) @ W0 + (dy.double() * U * sig) @ W1
    assert off(ops().int4_gated_backward(dy, u, v, p0, s0, p1, s1, gs), want) <= norm_bound(dt)


@pytest.mark.parametrize("T", [1, 20, 150, 700])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_block_norm_wise(T, dt):
    """Roundings of half a step on the way through the block, each h / sqrt(3) norm-wise: the norm's result, which reaches both
    projections (an elasticity of silu of 1.5 and one of 1: 1.8), the gated product, the stream, the result: 2.5 together."""
    from forge.inference import Int4FeedForward
    H, I, gs = 1024, 776, 64
    g = torch.Generator(device=DEV).manual_seed(T)
    mats = [matrix(I, H, gs, g), matrix(I, H, gs, g), matrix(H, I, gs, g)]
    x, res = (torch.randn(T, H, generator=g, device=DEV).to(dt) for _ in range(2))
    w = (1 + 0.2 * torch.randn(H, generator=g, device=DEV)).to(dt)
    blk = Int4FeedForward(*[m[:2] for m in mats], group_size=gs, norm_weight=w)
    h = x.double() + res.double()
    n = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6) * w.double()
    a = n @ mats[0][2].T
    want = (a * torch.sigmoid(a) * (n @ mats[1][2].T)) @ mats[2][2].T + h
    with torch.no_grad():
        assert off(blk(x, residual=res), want) <= 1.1 * 2.5 * HALF[dt] / math.sqrt(3)
    blk.check()


@pytest.mark.parametrize("T,C,R", [(2, 384, 22), (40, 1032, 700), (200, 520, 1001), (2600, 1000, 1000)])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_fp16_gradients_are_off_by_their_own_rounding(T, C, R, act):
    """dz and the weight rounded to 11 bits each would put the gradient off by sqrt(3) of its own rounding."""
    g = torch.Generator(device=DEV).manual_seed(T + C)
    p0, s0, W0 = matrix(R, C, 64, g)
    z = torch.randn(T, R, generator=g, device=DEV).half()
    dy = (torch.randn(T, R, generator=g, device=DEV) * torch.exp2(-8 * torch.rand(T, R, generator=g, device=DEV))).half()
    Z = z.double()
    sig = torch.sigmoid(Z)
    d = {"none": torch.ones_like(Z), "relu": (Z > 0).double(), "silu": sig * (1 + Z * (1 - sig)),
         "gelu": torch.special.ndtr(Z) + Z * torch.exp(-Z * Z / 2) / math.sqrt(2 * math.pi)}[act]
    dz = dy.double() * d
    dx, _ = ops().int4_linear_backward(dy, p0, s0, 64, preact=z, act=act)
    assert off(dx, dz @ W0) <= norm_bound(torch.float16)
