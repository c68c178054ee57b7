"""What Int4FeedForward keeps of the tensors that it is made from, and what it refuses.  No GPU: nothing is run on one."""
import io

import pytest
import torch

E, H, I, GS = 6, 128, 64, 32


def quantised(bits=4, symmetric=True, keep_codes=True, gs=GS):
    """A result of the layer quantiser, as far as the block reads it: codes, scales, zero points and packed words of E
    experts.  Asymmetric codes differ from their zero point by more than a nibble holds."""
    g = torch.Generator().manual_seed(3)
    out = {}
    for fam, R, C in (("gate", I, H), ("up", I, H), ("down", H, I)):
        q = torch.randint(0, 1 << bits, (E, R, C), generator=g, dtype=torch.uint8)
        z = torch.full((E, R, C // gs), float(1 << (bits - 1)))
        if not symmetric:
            z[..., 1] = 3.0
        nib = (q.to(torch.int64) - z.repeat_interleave(gs, 2).to(torch.int64) + 8).view(E, R, C // 8, 8) & 255
        words = (nib << (4 * torch.arange(8))).sum(-1)
        out[fam] = {"qweight": q if keep_codes else None, "scales": torch.rand(E, R, C // gs, generator=g) + 0.5, "qzeros": z,
                    "weight_packed": ((words + (1 << 31)) % (1 << 32) - (1 << 31)).to(torch.int32)}
    return out


def block(out, index=2, **kw):
    from forge.inference import Int4FeedForward
    return Int4FeedForward.from_quantized(out, index, **{"group_size": GS, **kw})


def test_a_block_of_a_batch_owns_its_matrices():
    out = quantised()
    blk = block(out)
    want = {n: b.clone() for n, b in blk.named_buffers()}
    for n, b in blk.named_buffers():
        assert b.untyped_storage().nbytes() == b.numel() * b.element_size(), n
    f = io.BytesIO()
    torch.save(blk.state_dict(), f)
    assert len(f.getvalue()) < sum(b.numel() * b.element_size() for b in want.values()) + 6000      # (the file's own records)
    for fam in ("gate", "up", "down"):
        out[fam]["weight_packed"].zero_()
        out[fam]["scales"].zero_()
    for n, b in blk.named_buffers():
        assert torch.equal(b, want[n]), n
    assert torch.equal(blk.gate_scales, quantised()["gate"]["scales"][2])
