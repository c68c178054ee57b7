"""GELU and its derivative where they are small: z Phi(z) for z down to -8.

Tolerances, derived before the first run, relative to the value.  A product with the weight matrix 1 (one code of one times a
scale of one) gives z = x exactly.  Phi(z) for z < 0 is exp(-z^2 / 2) times a smooth factor that is off by 2^-21; the exponent is
rounded twice, 2^-24 of it each, 2^-18 at z = -8, and the exponential is off by 2 + 1.17 z^2 / 2 units of 2^-23 at most (its
documented bound), 2^-17.7 there; the products 2^-22.  Together less than 2^-16, far below half a step of the result's type
(bf16 2^-8, fp16 2^-11), which is added; fp16 results below 2^-14 have steps of 2^-24, half of it 2^-25.  The derivative
Phi(z) + z phi(z) for z <= -2 is a difference of which the second term is at least four times the first, so an error of either
grows by 5/3 at most: 2^-15 covers both.  dz is then rounded to fp16 (2^-11) and W' = 1 is exact."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ops():
    from forge import ops as o
    return o


def identity(C, gs=32):
    """packed words and scales of the C x C matrix 1: code 9 on the diagonal, 8 elsewhere"""
    codes = torch.full((C, C), 8, dtype=torch.int64)
    codes.fill_diagonal_(9)
    w = (codes.view(C, C // 8, 8) << (4 * torch.arange(8))).sum(-1)
    return ((w + (1 << 31)) % (1 << 32) - (1 << 31)).to(torch.int32).to(DEV), torch.ones(C, C // gs, device=DEV)


def tail(T, C, dt):
    z = -(torch.arange(T * C, dtype=torch.float64) * 0.754877666 % 1) * 6 - 2          # -8 .. -2
    return z.view(T, C).to(dt).to(DEV)


@pytest.mark.parametrize("T,C", [(5, 64), (70, 64), (2600, 1024)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_gelu_of_negative_values(T, C, dt):
    packed, scales = identity(C)
    x = tail(T, C, dt)
    tiny = 2.0 ** -25 * (dt == torch.float16)
    y, z = ops().int4_linear(x, packed, scales, 32, act="gelu", want_preact=True)
    assert torch.equal(z, x)
    want = x.double() * torch.special.erfc(-x.double() / math.sqrt(2)) / 2
    assert bool(((y.double() - want).abs() <= (HALF[dt] + 2.0 ** -16) * want.abs() + tiny).all())
    # gated, times an up projection that is 1: a matrix whose row r sums x's channel 0, which holds 1
    x1 = x.clone()
    x1[:, 0] = 1
    up = torch.full_like(packed, -0x77777778)
    up[:, 0] = -0x77777778 + 1
    h = ops().int4_gated(x1, packed, scales, up, scales, 32, act="gelu")
    want = x1.double() * torch.special.erfc(-x1.double() / math.sqrt(2)) / 2
    assert bool(((h.double() - want).abs() <= (HALF[dt] + 2.0 ** -16) * want.abs() + tiny).all())


@pytest.mark.parametrize("T,C", [(5, 64), (5, 72), (2600, 1024)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_derivative_of_gelu_at_negative_values(T, C, dt):
    """Every token has one entry, so that its own power of two brings it into fp16's range whatever its size."""
    C8 = C // 8 * 8
    codes = torch.full((C8, C8), 8, dtype=torch.int64)
    codes.fill_diagonal_(9)
    packed, scales = (identity(C) if C % 32 == 0 else
                      ((((codes.view(C8, C8 // 8, 8) << (4 * torch.arange(8))).sum(-1) + (1 << 31)) % (1 << 32) - (1 << 31))
                       .to(torch.int32).to(DEV), torch.ones(C8, -(-C8 // 32), device=DEV)))
    z = tail(T, C8, dt)
    at = torch.arange(T, device=DEV) * 7 % C8
    lift = 256.0 if dt == torch.float16 else 1.0
    dy = torch.zeros(T, C8 + (C8 == 72), device=DEV, dtype=dt)[:, C8 == 72:]         # (72: rows that start off 16 bytes)
    dy[torch.arange(T, device=DEV), at] = lift
    dx, db = ops().int4_linear_backward(dy, packed, scales, 32, preact=z, act="gelu", want_dbias=True)
    Z = z.double()
    d = torch.special.erfc(-Z / math.sqrt(2)) / 2 + Z * torch.exp(-Z * Z / 2) / math.sqrt(2 * math.pi)
    want = dy.double() * d
    tiny = 2.0 ** -25 * (dt == torch.float16)
    assert bool(((dx.double() - want).abs() <= (HALF[dt] + 2.0 ** -11 + 2.0 ** -15) * want.abs() + tiny).all())
    total = want.sum(0)
    assert bool(((db.double() - total).abs() <= (HALF[dt] + 2.0 ** -15 + T * 2.0 ** -24) * want.abs().sum(0) + tiny).all())


@pytest.mark.parametrize("T", [7, 70])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_gelu_far_out(T, dt):
    """0 below, z above; in between, at -13 and in bf16, a normal number of 2^-123 (exponent and exponential are off by 2^-15)."""
    packed, scales = identity(64)
    at = torch.tensor([-6e4, -300.0, -40.0, -13.0, -0.0, 0.0, 13.0, 40.0, 300.0, 6e4], dtype=torch.float64)
    x = at.repeat(64)[:64].repeat(T, 1).to(dt).to(DEV)
    y = ops().int4_linear(x, packed, scales, 32, act="gelu").double()
    want = x.double() * torch.special.erfc(-x.double() / math.sqrt(2)) / 2
    assert bool(((y - want).abs() <= (HALF[dt] + 2.0 ** -14) * want.abs() + 2.0 ** -25 * (dt == torch.float16)).all())
    dy = torch.ones_like(x) / 64
    _, db = ops().int4_linear_backward(dy, packed, scales, 32, preact=x, act="gelu", want_dx=False, want_dbias=True)
    X = x[0].double()
    d = torch.special.erfc(-X / math.sqrt(2)) / 2 + X * torch.exp(-X * X / 2) / math.sqrt(2 * math.pi)
    assert bool(((db.double() - d * T / 64).abs() <= (HALF[dt] + 2.0 ** -14) * d.abs() * T / 64 + 2.0 ** -25 * (dt == torch.float16)).all())
