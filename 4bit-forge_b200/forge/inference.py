"""Inference over the packed sparse 1:4 + int4 experts: the runtime of the reference's sparse14_gemm.py:23-65
(Sparse14MoERuntime) on the grouped kernels.

The reference sorts the (token, slot) pairs by expert with vLLM's moe_permute, copies the hidden states into that
order and loops over experts and 256-row chunks with two per-expert GEMM calls and a torch SwiGLU between them.  Here
the sort is the routing-list kernel of the quantisation path, the permuted copy is replaced by a gather inside the
first kernel, and each projection pair is ONE launch over all experts (forge_sparse14_moe_w13_swiglu,
forge_sparse14_moe_w2).  Nothing is read back on the way.
"""
from __future__ import annotations

import torch

from . import _abi, ops


class Sparse14MoERuntime:
    """Same constructor and forward signature as sparse14_gemm.py:23-31.  w13_packed [E, G2(H), 2I, 2] and w2_packed
    [E, G2(I), H, 2] are the stacked outputs of the Wpair packer (uint64 bit patterns)."""

    def __init__(self, w13_packed, w2_packed, intermediate_size, num_experts, chunk_m=256):
        self.w13_packed = self._words(w13_packed)
        self.w2_packed = self._words(w2_packed)
        self.intermediate_size = int(intermediate_size)
        self.num_experts = int(num_experts)
        self.chunk_m = int(chunk_m)          # kept for signature compatibility; the grouped kernels need no chunking
        if self.w13_packed.shape[0] != self.num_experts or self.w2_packed.shape[0] != self.num_experts:
            raise RuntimeError("packed weights must be stacked over the experts")
        if self.w13_packed.shape[2] != 2 * self.intermediate_size:
            raise RuntimeError("w13_packed must hold 2 * intermediate_size rows (gate rows first)")
        self._active = torch.arange(self.num_experts, dtype=torch.int32, device=self.w13_packed.device)

    @staticmethod
    def _words(w):
        if not (w.dim() == 4 and w.shape[3] == 2):
            raise RuntimeError("packed weights must be [E, G2, R, 2]")
        w = w.contiguous()
        return w if w.dtype == torch.int64 else w.view(torch.int64)

    @torch.no_grad()
    def forward(self, hidden_states, topk_ids, topk_weights):
        """hidden_states bf16 [T, H], topk_ids [T, K], topk_weights [T, K] -> bf16 [T, H]: sum over the K slots of
        weight * down(silu(gate(x)) * up(x)) of the slot's expert (sparse14_gemm.py:32-65)."""
        T, H = hidden_states.shape
        K = topk_ids.shape[1]
        with torch.cuda.device(hidden_states.device):
            ids = topk_ids.to(torch.int32).contiguous()
            _, offsets, lists = ops.route_build_lists(ids, 0, self.num_experts)
            n = T * K
            a2 = ops.sparse14_moe_w13_swiglu(self.w13_packed, hidden_states, offsets, self._active, token_idx=lists,
                                             n_out=n)
            out_perm = ops.sparse14_moe_w2(self.w2_packed, a2, offsets, self._active, n_out=n)
            # weighted un-permute: the router weight of (token, expert) for every permuted position, fp32 sum, one
            # rounding
            tok = lists[:n].to(torch.int64)
            pos = torch.arange(n, device=hidden_states.device)
            expert = torch.searchsorted(offsets[1:].contiguous(), pos, right=True).clamp_(max=self.num_experts - 1)
            w = (topk_weights[tok].float() * (ids[tok].to(torch.int64) == expert[:, None])).sum(1)
            out = torch.zeros((T, H), dtype=torch.float32, device=hidden_states.device)
            out.index_add_(0, tok, out_perm.float() * w[:, None])
        return out.to(hidden_states.dtype)


# ---- dense feed-forward block on pack-quantized int4 weights ---------------------------------------------------------
class _RMSNorm(torch.autograd.Function):
    """(y, h): h is the stream behind the norm, x + residual, or x itself.  x comes back as an output so that the gradient
    that reaches it past the norm is added to the norm's own before that is rounded."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h = (ops.rmsnorm(x, weight, eps), x) if residual is None else ops.rmsnorm(x, weight, eps, residual=residual)
        ctx.save_for_backward(h, weight)
        ctx.eps, ctx.has_residual = eps, residual is not None
        return y, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        h, weight = ctx.saved_tensors
        dx, dw = ops.rmsnorm_backward(dy, h, weight, ctx.eps, dresidual=dh)
        return dx, dw, dx if ctx.has_residual else None, None


class _Int4Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, residual, packed, scales, gs, act, status):
        want = act != "none"
        out = ops.int4_linear(x, packed, scales, gs, bias=bias, act=act, residual=residual, want_preact=want,
                              status=status)
        y, z = out if want else (out, None)
        ctx.save_for_backward(z, packed, scales)
        ctx.gs, ctx.act, ctx.status = gs, act, status
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        z, packed, scales = ctx.saved_tensors
        need_x, need_b, need_r = ctx.needs_input_grad[:3]
        dx = db = None
        if need_x or need_b:
            dx, db = ops.int4_linear_backward(dy, packed, scales, ctx.gs, preact=z, act=ctx.act, want_dx=need_x,
                                              want_dbias=need_b, status=ctx.status)
        return dx, db, dy if need_r else None, None, None, None, None, None


class _Int4Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, sg, wu, su, gs, act, status):
        h, g, u = ops.int4_gated(x, wg, sg, wu, su, gs, act=act, want_preact=True, status=status)
        ctx.save_for_backward(g, u, wg, sg, wu, su)
        ctx.gs, ctx.act, ctx.status = gs, act, status
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        g, u, wg, sg, wu, su = ctx.saved_tensors
        dx = ops.int4_gated_backward(dh, g, u, wg, sg, wu, su, ctx.gs, act=ctx.act, status=ctx.status)
        return dx, None, None, None, None, None, None, None


def _grad_wanted(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class Int4FeedForward(torch.nn.Module):
    """The dense feed-forward block on the quantiser's own results: a shared expert, or any gated block whose three
    matrices went through pack_int4 with symmetric codes.

        forward(hidden)            -> down(act(gate(x)) * up(x)) [+ hidden],   x = norm(hidden)
        forward(hidden, residual)  -> the same with hidden + residual in hidden's place

    gate, up [I, H/8] and down [H, I/8] are (weight_packed, scales) pairs, kept as they are given where they are contiguous
    (and the scales fp32).  With norm_weight [H] the block starts with a root-mean-square norm and its result is added to the
    residual stream (three kernels: norm, gated product, product with the residual in its epilogue); without one it is the
    bare block and takes no residual.  The int4 weights are frozen; gradients reach hidden, residual and the norm's gain
    (tuning through the quantised block).  `status` (int32, on the block's device, not part of the state dict) collects what
    the kernels report; check() reads it.  The reference runs its packed dense experts through vLLM and has no such block of
    its own."""

    def __init__(self, gate, up, down, group_size=128, act="silu", norm_weight=None, eps=1e-6):
        super().__init__()
        self.group_size, self.act, self.eps = int(group_size), act, float(eps)
        gs = self.group_size
        if gs not in (32, 64, 128) or act not in _abi.ACTS:
            raise RuntimeError(f"group size must be 32, 64 or 128 and act one of {', '.join(_abi.ACTS)}")
        for name, (packed, scales) in (("gate", gate), ("up", up), ("down", down)):
            if packed.dim() != 2 or packed.dtype != torch.int32:
                raise RuntimeError(f"{name} must be packed words, int32 [R, C/8], got {packed.dtype} {list(packed.shape)}")
            want = (packed.shape[0], -(-packed.shape[1] * 8 // gs))
            if scales.shape != want:
                raise RuntimeError(f"the scales of {name} must be [R, ceil(C/{gs})] = {list(want)}, got {list(scales.shape)}")
            self.register_buffer(name + "_packed", packed.contiguous())
            self.register_buffer(name + "_scales", scales.to(torch.float32).contiguous())
        I, H8 = self.gate_packed.shape
        if self.up_packed.shape != (I, H8) or self.down_packed.shape != (H8 * 8, I // 8) or I % 8:
            raise RuntimeError("gate and up must be [I, H/8] and down [H, I/8] packed words")
        if norm_weight is not None and norm_weight.shape != (H8 * 8,):
            raise RuntimeError(f"norm_weight must be [{H8 * 8}], got {list(norm_weight.shape)}")
        self.norm_weight = None if norm_weight is None else torch.nn.Parameter(norm_weight.detach().clone())
        self.status = torch.zeros(1, dtype=torch.int32, device=self.gate_packed.device)

    def check(self):
        """Raises when a kernel of an earlier call of this block, forward or backward, reported a failure (a bounded wait
        that ran out): what that call returned is not valid.  Reads one word from the device, so it waits for the calls
        on the current stream; it is left to the caller, once a step or once a request, and cannot be captured."""
        code = int(self.status)
        if code != 0:
            self.status.zero_()
            raise RuntimeError("forge.inference: " + ("a bounded device-side wait ran out (FORGE_ERR_TIMEOUT)"
                               if code == _abi.ERR_TIMEOUT else f"a kernel reported status {code}")
                               + "; results of this block since the last check are not valid")

    def _apply(self, fn, recurse=True):
        """Module.to(dtype), .half() and the like move the scales but leave them in fp32: they are part of the codes.  The
        status word goes with them to another device and stays where it is otherwise (captured graphs write to it)."""
        status, dev = self.status, self.gate_packed.device
        kept = {name: getattr(self, name) for name in ("gate_scales", "up_scales", "down_scales")}
        super()._apply(fn, recurse)
        for name, scales in kept.items():
            if getattr(self, name).dtype != torch.float32:
                setattr(self, name, scales.to(getattr(self, name).device))
        if self.gate_packed.device != dev:
            new = self.gate_packed.device
            self.status = torch.zeros(1, dtype=torch.int32, device=new) if dev.type == "meta" else status.to(new)
        return self

    @classmethod
    def from_quantized(cls, out, index, group_size=128, **kw):
        """Matrix `index` of every family of MoELayerQuantizer.quantize_experts(...) (cfg.pack, symmetric, "gptq"): routed
        experts first, then the shared ones.  The block copies its matrices out of the batch.  Codes that the packed words
        do not hold (asymmetric ones, more than 4 bits) are refused."""
        pairs = []
        for fam in ("gate", "up", "down"):
            r = out[fam]
            if "weight_packed" not in r:
                raise RuntimeError(f"{fam} holds no packed int4 words: quantise with pack=True and algorithm 'gptq'")
            packed = r["weight_packed"][index].clone()
            scales = r["scales"][index].reshape(packed.shape[0], -1).to(torch.float32, copy=True)
            pairs.append((packed, scales))
        block = cls(*pairs, group_size=group_size, **kw)
        for fam in ("gate", "up", "down"):
            if not cls._nibbles_hold(out[fam], index, block.group_size):
                raise RuntimeError(f"the codes of {fam} cannot be read back from its packed words: they are not symmetric "
                                   "codes of 4 bits or fewer")
        return block

    @staticmethod
    def _nibbles_hold(result, index, group_size):
        """Whether every code of the matrix is within -8 .. 7 of its zero point, so that its nibble is the code's own: from
        the codes where the result keeps them, else for zero points that are all those of symmetric codes of 2, 3 or 4
        bits.  One read by the host."""
        z, q = result["qzeros"][index], result.get("qweight")
        if q is None:
            return any(torch.stack([(z == v).all() for v in (2, 4, 8)]).tolist())
        q = q[index]
        z = z.reshape(q.shape[0], -1).to(torch.int16).repeat_interleave(group_size, 1)[:, :q.shape[1]]
        d = q.to(torch.int16) - z
        return bool(((d >= -8) & (d <= 7)).all())

    def forward(self, hidden, residual=None):
        if residual is not None and self.norm_weight is None:
            raise RuntimeError("a block without a norm takes no residual")
        shape = hidden.shape
        if residual is not None and residual.shape != shape:
            raise RuntimeError(f"residual must have hidden's shape {list(shape)}, got {list(residual.shape)}")
        x = hidden.reshape(-1, shape[-1])
        res = None if residual is None else residual.reshape(-1, shape[-1])
        w, gs, act, status = self.norm_weight, self.group_size, self.act, self.status
        gate = (self.gate_packed, self.gate_scales, self.up_packed, self.up_scales, gs)
        down = (self.down_packed, self.down_scales, gs)
        if _grad_wanted(x, res, w):
            if w is None:
                y, h = x, None
            else:
                y, h = _RMSNorm.apply(x, w, res, self.eps)
            a = _Int4Gated.apply(y, *gate, act, status)
            out = _Int4Linear.apply(a, None, h, *down, "none", status)
        else:
            if w is None:
                y, h = x, None
            elif res is None:
                y, h = ops.rmsnorm(x, w, self.eps), x
            else:
                y, h = ops.rmsnorm(x, w, self.eps, residual=res)
            out = ops.int4_linear(ops.int4_gated(y, *gate, act=act, status=status), *down, residual=h, status=status)
        return out.view(shape)
