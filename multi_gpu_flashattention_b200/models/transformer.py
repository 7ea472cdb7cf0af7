"""A context-parallel transformer block whose attention is ring attention.

Each rank holds its token shard of the hidden states ([B, L, d_model], in the
RingLayout's local order). Projections, norms, the MLP and rotary position
embeddings are ordinary per-token PyTorch ops; rotary angles use the tokens'
GLOBAL positions from the layout, so a zigzag or striped shard computes
exactly what the unsharded model computes. Attention (causal, GQA) runs over
the process group with `ring_attention`.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.norm import rms_norm
from ..ops.paged import PagedKVCache
from ..ops.rotary import apply_rotary, rotary_frequencies
from ..parallel.api import ring_attention
from ..parallel.layouts import RingLayout


class RMSNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps

    def forward(self, x):
        xf = x.float()
        return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)).to(x.dtype) * self.weight


def rotary(x: torch.Tensor, positions: torch.Tensor, base: float = 10000.0) -> torch.Tensor:
    """Rotate pairs (x[..., i], x[..., i + D/2]) by position * base^(-2i/D).
    x [B, L, H, D], positions [L] (global token positions)."""
    D = x.shape[-1]
    inv = base ** (-torch.arange(0, D // 2, device=x.device, dtype=torch.float32) * 2 / D)
    ang = positions.to(x.device, torch.float32)[:, None] * inv[None, :]
    cos, sin = ang.cos()[None, :, None, :], ang.sin()[None, :, None, :]
    x1, x2 = x[..., : D // 2].float(), x[..., D // 2:].float()
    return torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1).to(x.dtype)


_INV_FREQ: dict = {}


def _frequencies(head_dim: int, device: torch.device) -> torch.Tensor:
    """rotary()'s frequencies on a device, float64 (made once, with a synchronous copy; a
    module's buffer would follow it to 16 bits)."""
    key = (head_dim, device)
    if key not in _INV_FREQ:
        with torch.inference_mode(False):  # training saves it for backward
            _INV_FREQ[key] = rotary_frequencies(head_dim, device=device)[0]
    return _INV_FREQ[key]


class RingAttentionBlock(nn.Module):
    """Pre-norm block: x + Attn(RMSNorm(x)); then + SwiGLU(RMSNorm(.)).

    fused_ops: the norms (the second with the attention's residual) and the rotary
    embeddings run on the kernels, for CUDA tensors; each rounds its result once, where
    the plain ops round between."""

    fused_ops = False  # of modules that were saved whole without one

    def __init__(self, d_model: int, n_heads: int, n_kv_heads: Optional[int] = None,
                 head_dim: int = 128, mlp_mult: int = 4, causal: bool = True,
                 fused_ops: bool = False):
        super().__init__()
        self.h, self.hkv = n_heads, n_kv_heads or n_heads
        self.d = head_dim
        self.causal = causal
        self.fused_ops = fused_ops
        self.norm1, self.norm2 = RMSNorm(d_model), RMSNorm(d_model)
        self.wq = nn.Linear(d_model, self.h * head_dim, bias=False)
        self.wk = nn.Linear(d_model, self.hkv * head_dim, bias=False)
        self.wv = nn.Linear(d_model, self.hkv * head_dim, bias=False)
        self.wo = nn.Linear(self.h * head_dim, d_model, bias=False)
        hidden = mlp_mult * d_model
        self.w1 = nn.Linear(d_model, hidden, bias=False)
        self.w3 = nn.Linear(d_model, hidden, bias=False)
        self.w2 = nn.Linear(hidden, d_model, bias=False)

    def forward(self, x: torch.Tensor, layout: RingLayout, rank: int = 0, group=None,
                backend: Optional[str] = None) -> torch.Tensor:
        B, L, _ = x.shape
        pos = layout.positions(rank)
        pos = torch.cat([pos, pos.new_zeros(L - pos.numel())]) if pos.numel() < L else pos
        fused = self.fused_ops and x.is_cuda
        h = rms_norm(x, self.norm1.weight, eps=self.norm1.eps) if fused else self.norm1(x)
        q = self.wq(h).view(B, L, self.h, self.d)
        k = self.wk(h).view(B, L, self.hkv, self.d)
        v = self.wv(h).view(B, L, self.hkv, self.d)
        if fused:
            q, k = apply_rotary(q, k, pos.to(x.device), _frequencies(self.d, x.device))
        else:
            q, k = rotary(q, pos), rotary(k, pos)
        a = ring_attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=self.causal,
                           group=group, layout=layout, backend=backend)
        a = self.wo(a.reshape(B, L, self.h * self.d).to(x.dtype))
        if fused:
            # under autocast the stream is wider than the branch
            h, x = rms_norm(a.to(x.dtype), self.norm2.weight, residual=x, eps=self.norm2.eps)
        else:
            x = x + a
            h = self.norm2(x)
        return x + self.mlp(h)

    def mlp(self, h: torch.Tensor) -> torch.Tensor:
        return self.w2(F.silu(self.w1(h)) * self.w3(h))


IGNORE_INDEX = -100


def shard_targets(ids: torch.Tensor, layout: RingLayout, rank: int) -> torch.Tensor:
    """Next-token targets of rank's shard, in the layout's local order.

    ids: the full sequence [B, S] (int64). The target of the token at global
    position p is ids[:, p + 1]; the last position and padding rows get
    IGNORE_INDEX. With zigzag or striped layouts the next token usually lives on
    another rank, so targets are cut from the full sequence on the host."""
    B, S = ids.shape
    nxt = torch.full_like(ids, IGNORE_INDEX)
    nxt[:, :-1] = ids[:, 1:]
    out = layout.shard(nxt, rank)
    n = layout.local_len(rank)
    out[:, n:] = IGNORE_INDEX
    return out


class RingTransformerLM(nn.Module):
    """Decoder-only language model with context-parallel ring attention.

    Each rank runs every layer on its own token shard (ids [B, L] in the
    layout's local order, padded to the layout's max_local_len); attention is
    the ring over `group`, everything else is per token. Parameters are
    replicated, so after `loss(...).backward()` the gradients are summed over
    the group (all-reduce, as in data parallelism) to give the unsharded
    model's gradients."""

    fused_ops = False  # of modules that were saved whole without one

    def __init__(self, vocab: int, d_model: int, n_layers: int, n_heads: int,
                 n_kv_heads: Optional[int] = None, head_dim: int = 128, mlp_mult: int = 4,
                 tie_embeddings: bool = True, fused_ops: bool = False):
        super().__init__()
        self.embed = nn.Embedding(vocab, d_model)
        self.fused_ops = fused_ops
        self.blocks = nn.ModuleList(
            RingAttentionBlock(d_model, n_heads, n_kv_heads, head_dim, mlp_mult, causal=True,
                               fused_ops=fused_ops)
            for _ in range(n_layers))
        self.norm = RMSNorm(d_model)
        self.head = nn.Linear(d_model, vocab, bias=False)
        # small embeddings (std 0.02): with the default N(0, 1) and tied weights the
        # initial logits would have std ~sqrt(d_model) and the first losses would be
        # far above ln(vocab)
        nn.init.normal_(self.embed.weight, std=0.02)
        if tie_embeddings:
            self.head.weight = self.embed.weight

    def forward(self, ids: torch.Tensor, layout: RingLayout, rank: int = 0, group=None,
                backend: Optional[str] = None) -> torch.Tensor:
        """Logits [B, L, vocab] of the local shard."""
        x = self.embed(ids)
        for blk in self.blocks:
            x = blk(x, layout, rank, group=group, backend=backend)
        h = rms_norm(x, self.norm.weight, eps=self.norm.eps) if self.fused_ops and x.is_cuda else self.norm(x)
        return self.head(h)

    def make_cache(self, pages: int, page_size: int, slots: int, max_tokens: int) -> PagedKVCache:
        """An empty paged cache for serve(), of the model's type and device."""
        w = self.embed.weight
        return PagedKVCache.allocate(len(self.blocks), pages, page_size, self.blocks[0].hkv,
                                     self.blocks[0].d, slots, max_tokens, dtype=w.dtype, device=w.device)

    def _check_served(self, ids: torch.Tensor, cache: PagedKVCache, max_seqlen: int) -> None:
        """What a layer would refuse, before the cache grows."""
        w, blk, k = self.embed.weight, self.blocks[0], cache.k
        if ids.dim() != 1 or max_seqlen < 0:
            raise ValueError(f"ids must be [tokens] and max_seqlen not negative, got {list(ids.shape)} and {max_seqlen}")
        if k.shape[0] < len(self.blocks) or tuple(k.shape[3:]) != (blk.hkv, blk.d) or \
                k.dtype != w.dtype or k.device != w.device:
            raise ValueError("the cache does not fit the model: see make_cache()")
        if blk.h % blk.hkv or blk.h // blk.hkv > 128:
            raise ValueError("heads must be a multiple of kv heads, up to 128 times")

    @torch.no_grad()
    def serve(self, ids: torch.Tensor, cache: PagedKVCache, slots: torch.Tensor,
              cu_seqlens: torch.Tensor, max_seqlen: int) -> torch.Tensor:
        """Logits [tokens, vocab] of the sequences' next tokens, on one GPU.

        ids [tokens] packs the new tokens of the sequences in `slots`: sequence b's are
        ids[cu_seqlens[b]:cu_seqlens[b + 1]], at most max_seqlen, the first of a prompt,
        a chunk of one, or single tokens. They join the cache and see all that it holds of
        their sequence (slots, cu_seqlens: int32 CUDA tensors). Rows outside every sequence
        hold nothing; those of a sequence that got no room in the cache, which stays as it
        was, are NaN. bfloat16 or float16 parameters, head_dim 64 or 128."""
        self._check_served(ids, cache, max_seqlen)
        pos = cache.reserve(slots, cu_seqlens, ids.numel())
        inv_freq = _frequencies(self.blocks[0].d, ids.device)
        x = self.embed(ids)
        h = rms_norm(x, self.blocks[0].norm1.weight, eps=self.blocks[0].norm1.eps)
        for i, blk in enumerate(self.blocks):
            q, k, v = (w(h).view(ids.numel(), n, blk.d)
                       for w, n in ((blk.wq, blk.h), (blk.wk, blk.hkv), (blk.wv, blk.hkv)))
            q, k = apply_rotary(q, k, pos, inv_freq)
            cache.write(i, k, v, slots, cu_seqlens)
            a = cache.attend(i, q, slots, cu_seqlens, max_seqlen)
            h, x = rms_norm(blk.wo(a.flatten(1)), blk.norm2.weight, residual=x, eps=blk.norm2.eps)
            after = self.blocks[i + 1].norm1 if i + 1 < len(self.blocks) else self.norm
            h, x = rms_norm(blk.mlp(h), after.weight, residual=x, eps=after.eps)
        h.masked_fill_(cache.refused(slots, cu_seqlens, ids.numel())[:, None], float("nan"))
        return self.head(h)

    def loss(self, ids: torch.Tensor, targets: torch.Tensor, layout: RingLayout, rank: int = 0,
             group=None, backend: Optional[str] = None) -> torch.Tensor:
        """Mean next-token cross entropy over every real token of the sequence:
        this shard's summed loss divided by the token count of all shards."""
        import torch.distributed as dist
        logits = self(ids, layout, rank, group=group, backend=backend)
        local = F.cross_entropy(logits.float().flatten(0, 1), targets.flatten(),
                                ignore_index=IGNORE_INDEX, reduction="sum")
        count = (targets != IGNORE_INDEX).sum().to(torch.float32)
        if dist.is_initialized() and dist.get_world_size(group) > 1:
            count = count.clone()
            dist.all_reduce(count, group=group)
        return local / count.clamp(min=1.0)
