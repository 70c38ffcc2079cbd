"""Transformer blocks for packed volumes: rows that hold the tokens of several samples (stacks of scans of any size, one after the other, padded at
the end), with rotary positions over several axes (stack, height, width) instead of the fixed 2-D table, attention that stays inside a
sample, and norms on both sides of every branch.

    y = norm1(x)
    x, y = x + gate1 * post1(attention(y)),  norm2(x)
    x, y = x + gate2 * post2(mlp(y)),        norm1 of the next block (x)

The counterpart of utils.Block / engine.EncoderFn for such rows; the reference has no packed form (its blocks: mirage/utils.py:162-262).  Like
there, parameters are fp32 nn.Parameters, products run on the bf16 GEMM kernels, the residual stream is fp32, and the backward pass OVERWRITES
the parameters' gradient buffers (arena.grad_buffer): nothing has to be zeroed, and a parameter takes part once per backward pass.
"""
from typing import Optional, Sequence

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import engine as E
from . import kernels as K
from .arena import follow, grad_buffer
from .utils import Linear, Mlp

BF16, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------------------------------------------------- positions
def grid_positions(sizes: Sequence[int], lead: int = 0, device=None) -> torch.Tensor:
    """int32 [lead + prod(sizes), len(sizes)]: raster order over `sizes` (stack, height, width; the last runs fastest), behind `lead` tokens at the
    origin (global tokens: rotary positions leave a token at the origin as it is)."""
    axes = torch.meshgrid(*[torch.arange(n) for n in sizes], indexing="ij")
    at = torch.stack([a.reshape(-1) for a in axes], dim=1)
    return torch.cat([torch.zeros(lead, len(sizes), dtype=at.dtype), at]).to(device=device, dtype=torch.int32)


def rotary_frequencies(sections: Sequence[int], theta: float = 100.0, device=None) -> torch.Tensor:
    """float64 [sum(sections)]: theta^(-i / n) for pair i of the n pairs of each axis (radians per position unit)."""
    return torch.cat([theta ** (-torch.arange(n, dtype=torch.float64) / n) for n in sections]).to(device)


# ------------------------------------------------------------------------------------------------- differentiable operators
def _anchor(params, device):
    """A leaf that ties a module's Function to the graph in its parameters' place (their gradients do not travel through autograd), or None where
    nothing is to be learnt.  Of its own for every call: a backward pass may be captured into a graph while another graph of the same
    parameters lives, whose accumulation nodes belong to the stream of their first use."""
    if torch.is_grad_enabled() and any(p.requires_grad for p in params):
        return torch.empty((), device=device, requires_grad=True)
    return None


def _learns(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _dense(g):
    """a gradient in one piece that starts on 16 bytes (autograd also hands over slices of larger ones, dense but anywhere)"""
    if g is None or (g.is_contiguous() and g.data_ptr() % 16 == 0):
        return g
    return g.clone(memory_format=torch.contiguous_format)


def _dense_heads(g):
    """a gradient as the kernels read it: heads in one piece, rows and heads on 16 bytes (autograd also hands over broadcast and sliced ones)"""
    if g is None or (g.stride(-1) == 1 and not any(s % 8 for s in g.stride()[:-1]) and g.data_ptr() % 16 == 0):
        return g
    return g.clone(memory_format=torch.contiguous_format)


_MOD_TENSORS = ("slopes", "pos_q", "pos_k", "doc_q", "doc_k", "prefix")


def _mod_parts(mod: Optional[K.ScoreMod]):
    """a ScoreMod as plain values and as tensors: these are saved like operands, so that a change between the two passes is an error"""
    if mod is None:
        return None, ()
    return (mod.cap, mod.causal), tuple(getattr(mod, n) for n in _MOD_TENSORS)


def _mod_whole(plain, tensors) -> Optional[K.ScoreMod]:
    return None if plain is None else K.ScoreMod(plain[0], causal=plain[1], **dict(zip(_MOD_TENSORS, tensors)))


def _finite_padding(x, mod: Optional[K.ScoreMod]):
    """x [B, N, dim] with zeros for padding's values that are not finite (documents that do not fit x are the attention's to refuse)"""
    docs = () if mod is None or mod.doc_q is None else (mod.doc_q, mod.doc_k)
    if not docs or any(d.shape != x.shape[:2] or d.device != x.device for d in docs):
        return x
    doc = docs[0] if docs[0] is docs[1] else torch.maximum(*docs)      # a token that only asks or only answers is no padding
    return torch.where((doc < 0).unsqueeze(-1), torch.nan_to_num(x, 0.0, 0.0, 0.0), x)


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, freqs, sections, pairing):
        ctx.save_for_backward(pos, freqs)
        ctx.how = (sections, pairing)
        return K.rotary_axes(q, k, pos, freqs, sections, pairing=pairing)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        pos, freqs = ctx.saved_tensors
        dq, dk = _dense_heads(dq), _dense_heads(dk)
        dq, dk = K.rotary_axes(dq, dk, pos, freqs, ctx.how[0], pairing=ctx.how[1], inverse=True)
        return dq, dk, None, None, None, None


def rotary(q, k, pos, freqs, sections, pairing: str = "axial"):
    """kernels.rotary_axes with its gradient (q and k of [B, N, heads, head_dim], bf16 or fp32)."""
    return _RotaryFn.apply(q, k, pos, freqs, tuple(sections), pairing)


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, mod, learns):
        o, saved = K.attn_mod_fwd(q, k, v, scale, mod, need_lse=learns)
        if learns:
            plain, tensors = _mod_parts(mod)
            ctx.save_for_backward(q, k, v, o, *saved, *tensors)
            ctx.how = (scale, plain)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o):
        q, k, v, o, lse, o_rest, *tensors = ctx.saved_tensors
        scale, plain = ctx.how
        grads = K.attn_mod_bwd(q, k, v, o, K.AttnSaved(lse, o_rest), _dense_heads(d_o), scale, _mod_whole(plain, tensors))
        return (*grads, None, None, None)


def attention(q, k, v, scale: float, mod: Optional[K.ScoreMod] = None):
    """kernels.attn_mod_fwd with its gradient: [B, Nq, H, hd] from bf16 q [B, Nq, H, hd] and k, v [B, Nk, Hk, hd]."""
    return _AttentionFn.apply(q, k, v, scale, mod, _learns(q, k, v))


class _SeamFn(torch.autograd.Function):
    """kernels.resid_norm_fwd; the gradients of a per-sample gate are returned, those of the parameters written into their buffers."""

    @staticmethod
    def forward(ctx, x, branch, gates, seam, pre, anchor):
        how = dict(gate=gates if gates is not None else seam.gate, alpha=seam.alpha, post=_wb(seam.post), pre=_wb(pre), kind=seam.kind, eps=seam.eps)
        x_new, y, stats = K.resid_norm_fwd(x, branch, **how)
        ctx.seam, ctx.pre = seam, pre
        ctx.save_for_backward(x_new, branch, gates, stats)
        return x_new, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dx_new, dy):
        x_new, branch, gates, stats = ctx.saved_tensors
        seam, pre = ctx.seam, ctx.pre
        named = [("post_weight", seam.post and seam.post.weight), ("post_bias", seam.post and seam.post.bias), ("pre_weight", pre and pre.weight),
                 ("pre_bias", pre and pre.bias)] + ([("gate", seam.gate)] if gates is None else [])
        into = {n: grad_buffer(p) for n, p in named if p is not None}
        dx, dbranch, grads = K.resid_norm_bwd(_dense(dx_new), None if pre is None else _dense(dy), x_new, branch, stats,
                                              gate=gates if gates is not None else seam.gate, alpha=seam.alpha, post=_wb(seam.post), pre=_wb(pre), kind=seam.kind,
                                              eps=seam.eps, grads={n: g for n, g in into.items() if g is not None})
        if gates is not None and seam.gate is not None and seam.gate.grad is not None:
            seam.gate.grad.zero_()                                # it took no part: what an earlier pass left is not this pass' gradient
        return dx, dbranch, grads["gate"] if gates is not None else None, None, None, None


def _wb(norm):
    return None if norm is None else (norm.weight, norm.bias)


# ------------------------------------------------------------------------------------------------------------- modules
class Norm(nn.Module):
    """weight and bias of a norm that a seam applies; kind "layer" (with bias) or "rms" (without)"""

    def __init__(self, dim: int, kind: str = "layer"):
        super().__init__()
        if kind not in ("layer", "rms"):
            raise ValueError(f"mirage_amd.packed.Norm: kind {kind!r} is neither 'layer' nor 'rms'")
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim)) if kind == "layer" else None


class Seam(nn.Module):
    """x' = alpha x + gate * post(branch), y = pre(x') in one kernel (kernels.resid_norm_fwd).  gate: a learnt row of channels (its initial value, or
    None for no gate); forward(gates=[samples, dim]) puts one row per sample in its place.  The gradients of gate and norms sum over all rows, padding
    among them: in training it has to be finite."""

    def __init__(self, dim: int, kind: str = "layer", post: bool = True, gate: Optional[float] = 1.0, alpha: float = 1.0, eps: float = 1e-6):
        super().__init__()
        self.kind, self.alpha, self.eps = kind, float(alpha), float(eps)
        self.post = Norm(dim, kind) if post else None
        self.gate = nn.Parameter(torch.full((dim,), float(gate))) if gate is not None else None

    def forward(self, x, branch, pre: Optional[Norm] = None, gates: Optional[torch.Tensor] = None):
        """(x', y); y is None without `pre`"""
        params = [p for m in (self, pre) if m is not None for p in m.parameters()]
        return _SeamFn.apply(x, branch, gates, self, pre, _anchor(params, x.device))


class _PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y16, att, pos, mod, need, anchor):
        B, N, _ = y16.shape
        for lin in (att.qkv, att.proj):
            follow(lin.weight)
        qkv, _, _ = E.lin_fwd(y16, att.qkv)
        heads = qkv.view(B, N, att.num_heads + 2 * att.num_kv_heads, att.head_dim)
        q, k, v = att.split(heads)
        freqs = None
        if att.sections is not None:                              # q and k are turned where the projection left them
            freqs = att.freqs(y16.device)
            K.rotary_axes(q, k, pos, freqs, att.sections, pairing=att.pairing, out_q=q, out_k=k)
        o, saved = K.attn_mod_fwd(q, k, v, att.scale, mod, need_lse=need)
        branch, _, _ = E.lin_fwd(o.view(B, N, -1), att.proj)
        if need:
            ctx.att = att
            ctx.plain, tensors = _mod_parts(mod)
            ctx.save_for_backward(y16, qkv, pos, freqs, o, *saved, *tensors)
        return branch

    @staticmethod
    @once_differentiable
    def backward(ctx, dbranch):
        y16, qkv, pos, freqs, o, lse, o_rest, *tensors = ctx.saved_tensors
        att = ctx.att
        B, N, _ = y16.shape
        d_o, _ = E.lin_bwd(_dense(dbranch), o.view(B, N, -1), att.proj)
        q, k, v = att.split(qkv.view(B, N, -1, att.head_dim))
        d_qkv = torch.empty_like(qkv)
        dq, dk, dv = att.split(d_qkv.view(B, N, -1, att.head_dim))
        K.attn_mod_bwd(q, k, v, o, K.AttnSaved(lse, o_rest), d_o.view(o.shape), att.scale, _mod_whole(ctx.plain, tensors), dq=dq, dk=dk, dv=dv)
        if att.sections is not None:
            K.rotary_axes(dq, dk, pos, freqs, att.sections, pairing=att.pairing, inverse=True, out_q=dq, out_k=dk)
        dy, _ = E.lin_bwd(d_qkv, y16, att.qkv)
        E.join_side_stream()
        return dy, None, None, None, None, None


class PackedAttention(nn.Module):
    """Self attention over packed rows: one projection to q (num_heads) and k, v (num_kv_heads each, shared by groups of query heads), rotary positions
    (sections: pairs per axis; None: no rotation), attention under `mod` (kernels.ScoreMod), output projection.  bf16 in, bf16 out.  The projections'
    gradients sum over all rows, padding among them: in training it has to be finite (PackedEncoder sees to that)."""

    def __init__(self, dim: int, num_heads: int, num_kv_heads: Optional[int] = None, sections: Optional[Sequence[int]] = None, theta: float = 100.0,
                 pairing: str = "axial", qkv_bias: bool = True):
        super().__init__()
        self.num_heads, self.num_kv_heads = num_heads, num_kv_heads or num_heads
        self.head_dim = dim // num_heads
        if dim % num_heads or self.head_dim not in (32, 64) or num_heads % self.num_kv_heads:
            raise NotImplementedError(f"mirage_amd.PackedAttention: {num_heads} heads ({self.num_kv_heads} for keys) of {dim} channels: head_dim must be 32 or 64, "
                                      "and the key heads must divide the query heads")
        self.scale = self.head_dim ** -0.5
        self.sections, self.theta, self.pairing = (None if sections is None else tuple(sections)), float(theta), pairing
        self.qkv = Linear(dim, (num_heads + 2 * self.num_kv_heads) * self.head_dim, bias=qkv_bias)
        self.proj = Linear(dim, dim)
        self._freqs = {}

    def freqs(self, device) -> torch.Tensor:
        """the rotary table on `device` (float64 whatever type the module's parameters are cast to), for the sections and theta that the module has now"""
        made_for = (device, tuple(self.sections), self.theta)
        if made_for not in self._freqs:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("mirage_amd.PackedAttention: run the module once before capturing it (its rotary table is made on the first call)")
            with torch.inference_mode(False):                     # kept for later calls, training ones among them, whose backward pass saves it
                self._freqs[made_for] = rotary_frequencies(self.sections, self.theta, device)
        return self._freqs[made_for]

    def split(self, heads):
        h, k = self.num_heads, self.num_kv_heads
        return heads[:, :, :h], heads[:, :, h:h + k], heads[:, :, h + k:]

    def forward(self, y16, pos: Optional[torch.Tensor] = None, mod: Optional[K.ScoreMod] = None):
        if y16.dtype != BF16 or y16.dim() != 3 or not y16.is_contiguous():
            raise ValueError(f"mirage_amd.PackedAttention: needs contiguous bf16 [B, N, dim] (a norm's output), got {y16.dtype} {tuple(y16.shape)}")
        if y16.numel() == 0:
            raise ValueError(f"mirage_amd.PackedAttention: {tuple(y16.shape)} holds no tokens (the projections' products take at least one)")
        if (pos is None) != (self.sections is None):
            raise ValueError("mirage_amd.PackedAttention: positions go with rotary sections")
        if y16.is_cuda and y16.device.index != torch.cuda.current_device():
            raise ValueError(f"mirage_amd.PackedAttention: input on {y16.device}, the projections run on the current device cuda:{torch.cuda.current_device()}")
        anchor = _anchor(self.parameters(), y16.device)
        return _PackedAttentionFn.apply(y16, self, pos, mod, anchor is not None or _learns(y16), anchor)


class _PackedMlpFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y16, mlp, need, anchor):
        for lin in (mlp.fc1, mlp.fc2):
            follow(lin.weight)
        act, _, pre = E.lin_fwd(y16, mlp.fc1, gelu=True, save_pre=need)
        branch, _, _ = E.lin_fwd(act, mlp.fc2)
        if need:
            ctx.mlp = mlp
            ctx.save_for_backward(y16, pre, act)
        return branch

    @staticmethod
    @once_differentiable
    def backward(ctx, dbranch):
        y16, pre, act = ctx.saved_tensors
        d_pre, _ = E.lin_bwd(_dense(dbranch), act, ctx.mlp.fc2, gelu_pre=pre)
        dy, _ = E.lin_bwd(d_pre, y16, ctx.mlp.fc1)
        E.join_side_stream()
        return dy, None, None, None


class PackedBlock(nn.Module):
    """Parameters of one block (module docstring); PackedEncoder runs them, because a block's last seam already applies the next block's first norm."""

    def __init__(self, dim: int, num_heads: int, mlp_ratio: float = 4.0, num_kv_heads: Optional[int] = None, sections: Optional[Sequence[int]] = None,
                 theta: float = 100.0, pairing: str = "axial", norm: str = "layer", post_norm: bool = True, gate: Optional[float] = 1.0, alpha: float = 1.0,
                 eps: float = 1e-6):
        super().__init__()
        self.norm1 = Norm(dim, norm)
        self.attn = PackedAttention(dim, num_heads, num_kv_heads, sections, theta, pairing)
        self.seam1 = Seam(dim, norm, post_norm, gate, alpha, eps)
        self.norm2 = Norm(dim, norm)
        self.mlp = Mlp(dim, int(dim * mlp_ratio))
        self.seam2 = Seam(dim, norm, post_norm, gate, alpha, eps)

    def forward(self, x, y16, following: Optional[Norm], pos=None, mod=None, gates=None):
        """one block from (x, norm1(x)): (x, following(x) or None).  gates: (attention's, mlp's) rows per sample, [samples, dim] each"""
        g1, g2 = gates if gates is not None else (None, None)
        x, y16 = self.seam1(x, self.attn(y16, pos, mod), self.norm2, g1)
        anchor = _anchor(self.mlp.parameters(), y16.device)
        return self.seam2(x, _PackedMlpFn.apply(y16, self.mlp, anchor is not None or _learns(y16), anchor), following, g2)


class PackedEncoder(nn.Module):
    """A stack of PackedBlocks with a final norm: forward(x fp32 [B, N, dim], pos, mod, gates) -> (x, norm(x) in bf16).  `mod` carries the documents of the
    packed rows (and whatever else its scores need).  Padding tokens (documents below zero) pass through the row-wise parts like any token, see nothing
    and are seen by nothing: what they hold reaches no other token.  Weight gradients sum over all rows, so in training the values of
    padding that are not finite are taken as zero; positions are finite everywhere."""

    def __init__(self, dim: int, depth: int, num_heads: int, **block):
        super().__init__()
        if depth < 1:
            raise ValueError("mirage_amd.PackedEncoder: depth must be at least 1")
        self.blocks = nn.ModuleList([PackedBlock(dim, num_heads, **block) for _ in range(depth)])
        norm, eps = block.get("norm", "layer"), block.get("eps", 1e-6)
        self.norm = Norm(dim, norm)
        self._first = Seam(dim, norm, post=False, gate=None, alpha=0.0, eps=eps)          # no parameters: x' = 0 x + x, y = norm1(x)

    def forward(self, x, pos: Optional[torch.Tensor] = None, mod: Optional[K.ScoreMod] = None, gates=None):
        """gates: per block (attention's, mlp's) rows per sample, or None (the blocks' learnt channel gates)"""
        if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in self.parameters())):
            x = _finite_padding(x, mod)
        x, y16 = self._first(x, x, self.blocks[0].norm1)
        for i, blk in enumerate(self.blocks):
            following = self.blocks[i + 1].norm1 if i + 1 < len(self.blocks) else self.norm
            x, y16 = blk(x, y16, following, pos, mod, None if gates is None else gates[i])
        return x, y16
