"""Int4FeedForward: equal calls give equal bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def parts(H, I, gs, g):
    out = []
    for R, C in ((I, H), (I, H), (H, I)):
        words = torch.randint(-2 ** 31, 2 ** 31, (R, C // 8), generator=g, device=DEV).to(torch.int32)
        out.append((words, (torch.rand(R, -(-C // gs), generator=g, device=DEV) + 0.5) / (5 * math.sqrt(C))))
    return out


@pytest.mark.parametrize("T", [1, 33, 600])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_no_residual_is_a_residual_of_zeros(T, dt):
    """The norm sees the same rows either way, so outputs and gradients are the same bits: the gradient of the stream past the
    norm is added to the norm's own in fp32 both times, not rounded before."""
    from forge.inference import Int4FeedForward
    g = torch.Generator(device=DEV).manual_seed(T)
    H, I, gs = 256, 192, 64
    w = (1 + 0.2 * torch.randn(H, generator=g, device=DEV)).to(dt)
    blk = Int4FeedForward(*parts(H, I, gs, g), group_size=gs, norm_weight=w)
    x, dout = (torch.randn(T, H, generator=g, device=DEV).to(dt) for _ in range(2))

    def step(**kw):
        blk.norm_weight.grad = None
        a = x.clone().requires_grad_()
        y = blk(a, **kw)
        y.backward(dout)
        return y.detach(), a.grad, blk.norm_weight.grad
    for got, want in zip(step(), step(residual=torch.zeros_like(x))):
        assert torch.equal(got, want)
    # the gain frozen, or the input
    blk.norm_weight.requires_grad_(False)
    a = x.clone().requires_grad_()
    blk(a).backward(dout)
    assert torch.equal(a.grad, step(residual=torch.zeros_like(x))[1])
    blk.norm_weight.requires_grad_(True)
    blk.norm_weight.grad = None
    y = blk(x)
    y.backward(dout)
    assert torch.equal(blk.norm_weight.grad, step()[2]) and x.grad is None
    blk.check()
