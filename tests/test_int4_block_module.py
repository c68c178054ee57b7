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


def test_codes_that_a_nibble_does_not_hold_are_refused():
    for keep in (True, False):
        with pytest.raises(RuntimeError, match="symmetric"):
            block(quantised(symmetric=False, keep_codes=keep))
        with pytest.raises(RuntimeError, match="symmetric"):
            block(quantised(bits=8, keep_codes=keep))
        for bits in (2, 3, 4):
            block(quantised(bits=bits, keep_codes=keep))
    # one zero point of one matrix, and only for the expert that has it
    for fam in ("gate", "up", "down"):
        out = quantised(keep_codes=False)
        out[fam]["qzeros"][2, 5, 1] = 7
        block(out, 1)
        with pytest.raises(RuntimeError, match=fam):
            block(out, 2)
    # an asymmetric matrix whose codes all lie within a nibble of their zero point reads back exactly
    out = quantised()
    out["up"]["qzeros"][2, 0, 0] = 5
    out["up"]["qweight"][2, 0, :GS] = 9
    block(out)
    # a sparse result, or one that was not packed
    out = quantised()
    del out["down"]["weight_packed"]
    with pytest.raises(RuntimeError, match="pack"):
        block(out)


def test_sizes_that_do_not_fit_are_refused_at_construction():
    from forge.inference import Int4FeedForward
    out = quantised()
    for kw in (dict(group_size=64), dict(group_size=128), dict(group_size=16), dict(group_size=0), dict(act="tanh"),
               dict(norm_weight=torch.ones(H + 1)), dict(norm_weight=torch.ones(1, H))):
        with pytest.raises(RuntimeError):
            block(out, **kw)
    parts = [(out[f]["weight_packed"][0], out[f]["scales"][0]) for f in ("gate", "up", "down")]
    Int4FeedForward(*parts, group_size=GS)
    for k in range(3):
        for bad in ((parts[k][0], parts[k][1][:, :-1]), (parts[k][0], parts[k][1].t()), (parts[k][0].long(), parts[k][1]),
                    (parts[k][0][0], parts[k][1])):
            with pytest.raises(RuntimeError):
                Int4FeedForward(*[bad if i == k else p for i, p in enumerate(parts)], group_size=GS)


class FakeOps:
    """Shapes of the operators, and the status word that each call was given."""

    def __init__(self):
        self.calls = []

    def rmsnorm(self, x, w, eps, residual=None):
        return x.clone() if residual is None else (x.clone(), x + residual)

    def rmsnorm_backward(self, dy, x, w, eps, dresidual=None):
        return dy.clone(), torch.zeros_like(w)

    def int4_linear(self, x, packed, scales, gs, bias=None, act="none", residual=None, want_preact=False, status=None):
        self.calls.append(("linear", status))
        return x.new_zeros(x.shape[0], packed.shape[0])

    def int4_gated(self, x, wg, sg, wu, su, gs, act="silu", want_preact=False, status=None):
        self.calls.append(("gated", status))
        h = x.new_zeros(x.shape[0], wg.shape[0])
        return (h, h.clone(), h.clone()) if want_preact else h

    def int4_linear_backward(self, dy, packed, scales, gs, preact=None, act="none", want_dx=True, want_dbias=False, status=None):
        self.calls.append(("linear backward", status))
        return dy.new_zeros(dy.shape[0], packed.shape[1] * 8), None

    def int4_gated_backward(self, dh, g, u, wg, sg, wu, su, gs, act="silu", status=None):
        self.calls.append(("gated backward", status))
        return dh.new_zeros(dh.shape[0], wg.shape[1] * 8)


def test_every_product_reports_to_the_status_word(monkeypatch):
    from forge import inference
    fake = FakeOps()
    monkeypatch.setattr(inference, "ops", fake)
    for kw in ({}, {"norm_weight": torch.ones(H)}):
        blk = block(quantised(), **kw)
        for grad in (False, True):
            fake.calls.clear()
            x = torch.zeros(3, H, requires_grad=grad)
            y = blk(x, residual=torch.zeros(3, H)) if kw else blk(x)
            want = {"linear", "gated"}
            if grad:
                y.sum().backward()
                want |= {"linear backward", "gated backward"}
            elif kw:
                assert y.requires_grad           # (through the gain)
            assert {name for name, _ in fake.calls} == want
            assert all(s is blk.status for _, s in fake.calls)
        blk.check()
        blk.status.fill_(3)                      # as a kernel leaves it
        with pytest.raises(RuntimeError, match="FORGE_ERR_TIMEOUT"):
            blk.check()
        blk.check()                              # reported once
        blk.status.fill_(2)
        with pytest.raises(RuntimeError, match="status 2"):
            blk.check()


def test_the_status_word_moves_with_the_block():
    import copy
    blk = block(quantised(), norm_weight=torch.ones(H))
    assert "status" not in blk.state_dict() and blk.status.dtype == torch.int32
    word = blk.status
    blk.half().to(torch.bfloat16).double()
    assert blk.status is word
    other = copy.deepcopy(blk)
    other.status.fill_(3)
    blk.check()
    meta = copy.deepcopy(blk).to("meta")
    assert meta.status.device.type == "meta"
    assert int(meta.to_empty(device="cpu").status) == 0


def test_a_residual_of_another_shape_is_refused(monkeypatch):
    """Also one of as many elements, whose rows would meet those of hidden in an order that its shape does not say."""
    from forge import inference
    monkeypatch.setattr(inference, "ops", FakeOps())
    blk = block(quantised(), norm_weight=torch.ones(H))
    x = torch.zeros(2, 3, H)
    assert blk(x, residual=torch.zeros(2, 3, H)).shape == x.shape
    for shape in ((3, 2, H), (6, H), (2, 6, H // 2), (1, 3, H), (H,)):
        with pytest.raises(RuntimeError, match="shape"):
            blk(x, residual=torch.zeros(shape))


def test_the_backward_workspace_holds_the_powers_of_every_block_of_rows():
    from forge import _abi
    lib = _abi.load_library()
    for T, C, R, gs, mats in ((1, 8, 1, 32, 1), (5, 776, 513, 32, 2), (4096, 7168, 2048, 128, 2), (3, 40000, 700, 32, 1)):
        K, G = mats * R, -(-C // gs)
        n = lib.forge_int4_backward_workspace_bytes(T, C, R, gs, mats)
        rest = T * 4 + K * G * 4 + K * 4 + -(-K // 512) * G * 4 + 64 * R * 4
        assert n >= T * (-(-K // 64) * 64) * 4 + rest              # high and low parts of dz
        for dtype, act in ((_abi.BF16, "gelu"), (_abi.F16, "none"), (_abi.F16, "relu"), (_abi.F16, "silu")):
            m = lib.forge_int4_backward_workspace_bytes_for(dtype, _abi.ACTS[act], T, C, R, gs, mats)
            low = dtype == _abi.F16 and (mats == 2 or act == "silu")
            assert m == n if low else T * (-(-K // 64) * 64) * 2 + rest <= m <= n
    assert lib.forge_int4_backward_workspace_bytes_for(_abi.F16, 0, 1, 8, 8, 0, 1) == 0
