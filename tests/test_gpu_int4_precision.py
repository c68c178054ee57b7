"""How exact the backward products over packed int4 weights are: single sums with a known rounding, and norm-wise bounds.

Tolerances, derived before the first run.  A sum over k of terms with independent signs has a norm of the root of the sum of
the terms' squares, and so has the sum of their independent errors: a relative rounding of half a step h of every term
contributes h / sqrt(3) at most, norm-wise (an error spread evenly over the step).  dz is rounded to fp16 (2^-11), the weight
is rounded to fp16 (2^-11), and the result to its own type: sqrt((h_type^2 + 2 (2^-11)^2) / 3), and a tenth more for the
spread of the norms of a few thousand entries and the fp32 sums."""
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
    return 1.1 * math.sqrt((HALF[dt] ** 2 + 2 * 2.0 ** -22) / 3)


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
