"""Qwen3-8B-shaped prefill with every linear replaced by the W4A4 group-128 linear
(36 layers, hidden 4096, 32 query / 8 KV heads, head_dim 128, SwiGLU 12288,
RMSNorm, RoPE; attention stays in bf16 through torch SDPA).  Random-initialised weights: this is a
throughput harness for the caller side of the op boundary, not a checkpoint loader.

Decoding: ``prefill`` fills a paged cache (``DecodeCache``), ``step`` takes one token, a chain or a tree of drafts of every sequence
through the same packed weights with 16-bit activations, and ``commit`` keeps the accepted ones.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd import forward_ad
from torch.overrides import _get_current_function_mode_stack
from torch.utils._device import DeviceContext

from . import moe as _moe
from . import ops
from .linear import W4A4Linear, apply_quantized


@dataclass
class Qwen3Config:
    hidden: int = 4096
    layers: int = 36
    q_heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    inter: int = 12288
    vocab: int = 151936
    rope_theta: float = 1.0e6
    eps: float = 1e-6


def _plain(*tensors, align: int = 16) -> bool:
    """Whether an op that reads raw pointers may stand in for torch ops on these tensors: contiguous bf16 on one GPU, and
    nothing at work (a tracer, a mode, a functional transform, autograd in either direction) that has to see torch ops."""
    if torch.compiler.is_compiling() or torch.jit.is_tracing():
        return False
    if (forward_ad._current_level >= 0 or torch._C._functorch.peek_interpreter_stack() is not None
            or torch._C._len_torch_dispatch_stack() or any(type(m) is not DeviceContext for m in _get_current_function_mode_stack())):
        return False
    for t in tensors:
        if (type(t) not in (torch.Tensor, nn.Parameter) or not t.is_cuda or t.device != tensors[0].device
                or t.dtype != torch.bfloat16 or not t.is_contiguous() or t.is_neg() or t.data_ptr() % align
                or (t.requires_grad and torch.is_grad_enabled())):
            return False
    return True


class RMSNorm(nn.Module):
    def __init__(self, dim: int, eps: float, device=None):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim, dtype=torch.bfloat16, device=device), requires_grad=False)
        self.eps = eps

    def forward(self, x):
        if _plain(x, self.weight) and x.dim() > 0 and self.weight.shape == x.shape[-1:]:
            K = x.shape[-1]
            if K % 8 == 0 and 1024 <= K <= 16384 and x.numel() < K << 31:
                return ops.rmsnorm(x, self.weight, self.eps)
        xf = x.float()
        return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)).to(x.dtype) * self.weight


def _untouched(norm) -> bool:
    """An RMSNorm of this file that nobody hooked or patched: calling it is its expression and nothing else."""
    g = nn.modules.module
    return (type(norm) is RMSNorm and "forward" not in vars(norm)
            and not (norm._forward_hooks or norm._forward_pre_hooks or norm._backward_hooks or norm._backward_pre_hooks
                     or g._global_forward_hooks or g._global_forward_pre_hooks or g._global_backward_hooks
                     or g._global_backward_pre_hooks))


def rope_tables(seq: int, head_dim: int, theta: float, device):
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim))
    ang = torch.outer(torch.arange(seq, device=device, dtype=torch.float32), inv)
    return ang.cos().to(torch.bfloat16), ang.sin().to(torch.bfloat16)


def apply_rope(x, cos, sin):
    # x [B, H, S, D]; rotate-half convention
    d = x.shape[-1] // 2
    x1, x2 = x[..., :d], x[..., d:]
    c, s = cos[None, None], sin[None, None]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


def _bare(*linears) -> bool:
    """Whether these linears are their product and nothing else: no smoothing factors for the inputs, no bias."""
    return all(lin.smooth_scale is None and lin.bias is None for lin in linears)


class Block(nn.Module):
    def __init__(self, cfg: Qwen3Config, device, per_channel: bool, gen: torch.Generator, fused: bool = True):
        super().__init__()
        self.cfg = cfg
        qkv_out = (cfg.q_heads + 2 * cfg.kv_heads) * cfg.head_dim
        self.qkv = self._lin(cfg.hidden, qkv_out, device, per_channel, gen)
        self.o = self._lin(cfg.q_heads * cfg.head_dim, cfg.hidden, device, per_channel, gen)
        self.gate_up = self._lin(cfg.hidden, 2 * cfg.inter, device, per_channel, gen)
        self.down = self._lin(cfg.inter, cfg.hidden, device, per_channel, gen)
        self.ln1 = RMSNorm(cfg.hidden, cfg.eps, device)
        self.ln2 = RMSNorm(cfg.hidden, cfg.eps, device)
        self.q_norm = RMSNorm(cfg.head_dim, cfg.eps, device)
        self.k_norm = RMSNorm(cfg.head_dim, cfg.eps, device)
        # fold the quantisers into RMSNorm / SwiGLU (per-group scales only; the per-channel ops keep the plain path)
        self.fused = fused and not per_channel

    @staticmethod
    def _lin(k, n, device, per_channel, gen):
        lin = W4A4Linear(k, n, per_channel=per_channel, device=device)
        # fill in slabs so that an 8-billion-parameter model never needs an fp32 copy of a whole matrix
        for r0 in range(0, n, 4096):
            r1 = min(n, r0 + 4096)
            lin.weight.data[r0:r1] = (torch.randn(r1 - r0, k, device=device, generator=gen) * 0.02).to(torch.bfloat16)
        return lin.quantize_()  # the bf16 weight is released here

    def forward(self, x, cos, sin, attend=None):
        cfg = self.cfg
        B, S, _ = x.shape
        folded = self.qkv, self.gate_up, self.down     # (as they are now: a layer may have been given others)
        if self.fused and _bare(*folded) and all(lin.method.act_bits == 4 for lin in folded):
            return self._forward_fused(x, cos, sin, attend)
        qkv = self.qkv(self.ln1(x))
        if attend is not None:
            return self._feed_forward(x + self.o(attend(self, qkv)))
        q, k, v = qkv.split([cfg.q_heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim], -1)
        q = self.q_norm(q.view(B, S, cfg.q_heads, cfg.head_dim)).transpose(1, 2)
        k = self.k_norm(k.view(B, S, cfg.kv_heads, cfg.head_dim)).transpose(1, 2)
        v = v.view(B, S, cfg.kv_heads, cfg.head_dim).transpose(1, 2)
        q, k = apply_rope(q, cos, sin), apply_rope(k, cos, sin)
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
        return self._feed_forward(x + self.o(a.transpose(1, 2).reshape(B, S, -1)))

    def _feed_forward(self, x):
        gu = self.gate_up(self.ln2(x))
        g, u = gu.split(self.cfg.inter, -1)
        return x + self.down(F.silu(g) * u)

    def _turned_heads(self, qkv, positions, freqs):
        """Query, key and value heads [tokens, heads, head_dim] of qkv [tokens, width], normed and at their positions."""
        cfg = self.cfg
        q, k, v = qkv.view(qkv.shape[0], -1, cfg.head_dim).split([cfg.q_heads, cfg.kv_heads, cfg.kv_heads], 1)
        return ops.rope_(self.q_norm(q), positions, freqs), ops.rope_(self.k_norm(k), positions, freqs), v

    def step(self, x, positions, freqs, attend):
        """x [B, T, hidden] through the layer with 16-bit activations and ``attend(q, k, v)`` over [B, T, heads, head_dim]."""
        cfg = self.cfg
        B, T, H = x.shape

        def linear(lin, y):
            if lin.smooth_scale is not None:
                y = y / lin.smooth_scale.to(y.dtype)
            y = ops.w4a16_linear(y, lin.weight_int4, lin.weight_scale, lin.out_features, lin.method.per_channel)
            return y if lin.bias is None else y + lin.bias

        heads = self._turned_heads(linear(self.qkv, self.ln1(x).view(B * T, H)), positions, freqs)
        a = attend(*(t.unflatten(0, (B, T)) for t in heads))
        x = x + linear(self.o, a.view(B * T, -1)).view(B, T, H)
        y = self.ln2(x).view(B * T, H)
        if _bare(self.gate_up):
            up = ops.w4a16_gated_linear(y, self.gate_up.weight_int4, self.gate_up.weight_scale, cfg.inter, self.gate_up.method.per_channel)
        else:
            gate, up = linear(self.gate_up, y).split(cfg.inter, -1)
            up = F.silu(gate) * up
        return x + linear(self.down, up).view(B, T, H)

    def _attention(self, qkv, B, S, cos, sin):
        cfg = self.cfg
        # norms and rotary embedding in one kernel, in place (qkv is this layer's own buffer), where they are what they were
        # built as; else through the modules
        fused = (cfg.head_dim == 128 and _untouched(self.q_norm) and _untouched(self.k_norm)
                 and self.q_norm.eps == self.k_norm.eps and qkv.numel() > 0
                 and _plain(qkv, self.q_norm.weight, self.k_norm.weight, cos, sin, align=8)
                 and self.q_norm.weight.shape == self.k_norm.weight.shape == (128,) and cos.shape == sin.shape == (S, 64))
        if fused:
            ops.qk_norm_rope_(qkv.view(B * S, -1), self.q_norm.weight, self.k_norm.weight, cos, sin, cfg.q_heads,
                              cfg.kv_heads, S, self.q_norm.eps)
        q, k, v = qkv.split([cfg.q_heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim], -1)
        q, k, v = (t.view(B, S, -1, cfg.head_dim) for t in (q, k, v))
        if not fused:
            q, k = self.q_norm(q), self.k_norm(k)
        q, k, v = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
        if not fused:
            q, k = apply_rope(q, cos, sin), apply_rope(k, cos, sin)
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
        return a.transpose(1, 2).reshape(B, S, -1)

    def _forward_fused(self, x, cos, sin, attend=None):
        """Per-group mode with the quantisers folded into the ops in front of them: RMSNorm + quantise in one
        kernel before qkv and gate+up, SwiGLU + quantise in one kernel before down."""
        B, S, H = x.shape
        M = B * S
        xp, xs = ops.rmsnorm_int4_quant_grouped(x.view(M, H), self.ln1.weight, self.ln1.eps)
        qkv = apply_quantized(self.qkv, xp, xs, M).view(B, S, -1)
        x = x + self.o(self._attention(qkv, B, S, cos, sin) if attend is None else attend(self, qkv))
        xp, xs = ops.rmsnorm_int4_quant_grouped(x.view(M, H), self.ln2.weight, self.ln2.eps)
        gu = apply_quantized(self.gate_up, xp, xs, M)
        ap, asc = _moe.moe_silu_mul_quant(gu)
        return x + apply_quantized(self.down, ap, asc, M).view(B, S, H)


class DecodeCache:
    """Paged keys and values of a batch: ``k`` and ``v`` hold [pages, page_size, kv_heads, head_dim] for each layer, a sequence's pages
    are in ``block_table`` [batch, width] and its tokens counted in ``lengths`` [batch] (int32, on the device).  Here every sequence
    owns its pages from the start; a server hands them out by writing the table."""

    def __init__(self, cfg: Qwen3Config, batch: int, tokens: int, page_size: int = 64, device="cuda"):
        width = -(-tokens // page_size)
        shape = (batch * width, page_size, cfg.kv_heads, cfg.head_dim)
        self.k, self.v = ([torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(cfg.layers)] for _ in range(2))
        self.block_table = torch.arange(batch * width, dtype=torch.int32, device=device).view(batch, width)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.freqs = ops.rope_frequencies(cfg.head_dim, cfg.rope_theta, device)[0]
        self.pending: list = []       # keys and values of the last step, layer by layer, not yet in the cache

    def append(self, layer: int, k, v, counts=None, select=None) -> None:
        ops.kv_cache_append_(self.k[layer], self.v[layer], k, v, self.block_table, self.lengths, select=select, counts=counts)

    def accepted(self, tokens: int, counts: torch.Tensor | None = None, select: torch.Tensor | None = None, prompt: bool = False) -> torch.Tensor:
        """[batch] int32: how many of `tokens` new rows each sequence takes, all of ``counts[b]`` (all rows without), or -1 where it can take them
        not at all: a count or an index of ``select`` out of range, no room, a page that the table does not name, or (``prompt``) tokens for a
        sequence that is not empty.  An append with -1 writes nothing and is raised by ``ops.check_status``; nothing here waits
        for the device."""
        B, width = self.block_table.shape
        dev = self.lengths.device
        if counts is None:
            counts = torch.full_like(self.lengths, tokens)
        elif counts.dtype != torch.int32 or counts.shape != (B,) or counts.device != dev:
            raise RuntimeError("counts must be int32 [batch], on the cache's device")
        row = torch.arange(tokens, device=dev)
        at = self.lengths.long()[:, None] + row
        page_size = self.k[0].shape[1]
        fits = (at >= 0) & (at < width * page_size)
        if width:
            page = self.block_table.gather(1, (at // page_size).clamp(0, width - 1))
            fits &= (page >= 0) & (page < self.k[0].shape[0])
        if select is not None:
            if select.dtype != torch.int32 or select.dim() != 2 or select.shape[0] != B or select.shape[1] < tokens or select.device != dev:
                raise RuntimeError("select must be int32 [batch, new rows], on the cache's device")
            fits &= (select[:, :tokens] >= 0) & (select[:, :tokens] < tokens)
        ok = (fits | (row >= counts[:, None])).all(1) & (counts >= 0) & (counts <= tokens)
        if prompt:
            ok &= (self.lengths == 0) | (counts == 0)
        return torch.where(ok, counts, -1)

    def commit(self, counts: torch.Tensor | None = None, select: torch.Tensor | None = None) -> None:
        """Keeps ``counts[b]`` tokens of the last step (all without): its first ones, or rows ``select[b, :counts[b]]``, the accepted path of a
        tree.  int32; nothing waits for the device.  A sequence that cannot take its tokens (``accepted``) keeps its length and its
        cache, which ``ops.check_status`` raises."""
        if not self.pending:
            raise RuntimeError("commit: there is no step to keep tokens of")
        counts = self.accepted(self.pending[0][0].shape[1], counts, select)
        for layer, (k, v) in enumerate(self.pending):
            self.append(layer, k, v, counts, select)
        self.lengths += counts.clamp(min=0)
        self.pending = []


class Qwen3Prefill(nn.Module):
    def __init__(self, cfg: Qwen3Config = Qwen3Config(), device="cuda", per_channel: bool = False, seed: int = 1,
                 fused: bool = True):
        super().__init__()
        self.cfg = cfg
        gen = torch.Generator(device=device).manual_seed(seed)
        self.embed = nn.Embedding(cfg.vocab, cfg.hidden, device=device, dtype=torch.bfloat16)
        self.blocks = nn.ModuleList(Block(cfg, device, per_channel, gen, fused) for _ in range(cfg.layers))
        self.norm = RMSNorm(cfg.hidden, cfg.eps, device)

    @torch.no_grad()
    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        """Token ids [B, S] -> final hidden states [B, S, hidden] (prefill; no LM head, no KV cache)."""
        x = self.embed(ids)
        cos, sin = rope_tables(ids.shape[1], self.cfg.head_dim, self.cfg.rope_theta, ids.device)
        for blk in self.blocks:
            x = blk(x, cos, sin)
        return self.norm(x)

    @torch.no_grad()
    def prefill(self, ids: torch.Tensor, cache: DecodeCache, counts: torch.Tensor | None = None) -> torch.Tensor:
        """As ``forward`` for prompts [B, S] of which ``counts[b]`` tokens count (int32; all without), whose keys and values go into the empty
        sequences of ``cache``; a sequence without such tokens is left as it is.  One that cannot take its tokens (``DecodeCache.accepted``),
        because it is not empty for instance, stays as it was too, which ``ops.check_status`` raises."""
        cache.pending = []     # a step before the prompt is none behind it
        B, S = ids.shape
        freqs = cache.freqs
        positions = torch.arange(S, device=ids.device).repeat(B)
        counts = cache.accepted(S, counts, prompt=True)
        x = self.embed(ids)
        for layer, blk in enumerate(self.blocks):
            def attend(blk, qkv, layer=layer):
                q, k, v = (t.unflatten(0, (B, S)) for t in blk._turned_heads(qkv.reshape(B * S, -1), positions, freqs))
                cache.append(layer, k, v, counts)
                a = F.scaled_dot_product_attention(*(t.transpose(1, 2) for t in (q, k, v)), is_causal=True, enable_gqa=True)
                return a.transpose(1, 2).reshape(B, S, -1)

            x = blk(x, None, None, attend)
        cache.lengths += counts.clamp(min=0)
        return self.norm(x)

    @torch.no_grad()
    def step(self, ids: torch.Tensor, cache: DecodeCache, tree_mask: torch.Tensor | None = None) -> torch.Tensor:
        """One token, a chain or a tree of drafts of every sequence: ids [B, T] -> final hidden states [B, T, hidden].  In a tree node t sees
        the nodes j with ``tree_mask[b, t, j]`` (bool, itself and its ancestors) and stands that many positions behind the cache.
        ``cache.commit`` keeps the accepted ones; until then the cache is as it was, and the next ``step`` forgets them.  A captured graph
        holds a step with its ``commit``: a replay leaves nothing to commit."""
        cache.pending, made = [], []     # a step that raises half-way leaves nothing to commit
        B, T = ids.shape
        freqs = cache.freqs
        if tree_mask is None:
            depth = torch.arange(T, device=ids.device)
        else:
            depth = tree_mask.sum(-1) - 1
        positions = (cache.lengths[:, None] + depth).flatten()
        x = self.embed(ids)
        for layer, blk in enumerate(self.blocks):
            def attend(q, k, v, layer=layer):
                made.append((k, v))
                return ops.tree_attention(q, k, v, cache.k[layer], cache.v[layer], cache.block_table, cache.lengths, tree_mask=tree_mask)

            x = blk.step(x, positions, freqs, attend)
        x = self.norm(x)
        cache.pending = made
        return x
