"""B200-native ring attention.

Public API
----------
ring_attention(q, k, v, causal=False, group=None, layout=None, ...)
    Context-parallel attention over a torch.distributed group; each rank holds
    its token shard of q, k, v ([batch, local_seq, heads, head_dim]).
RingLayout(kind, seq, world)
    contiguous / zigzag / striped / scheduler-driven token ownership.
flash_attn(q, k, v, causal=False, softmax_scale=None)
    Single-GPU attention on the sm_100a kernels (differentiable);
    flash_attn_fwd / flash_attn_bwd are the explicit passes.
GraphedAttention(q, k, v, causal=False, backward=False)
    The single-GPU passes captured into CUDA graphs for fixed shapes.
rms_norm(x, weight, residual=None), rms_norm_fp8(...)
    Root-mean-square norm with the residual's addition (differentiable), and its
    output in 8 bits with scales.
apply_rotary(q, k, positions, inv_freq), rotary_frequencies(rotary_dim, ...)
    Rotary positions in both layouts (differentiable), and their (scaled) frequencies.
apply_norm_rotary(q, k, positions, inv_freq, q_weight, k_weight)
    The same behind a root-mean-square norm of each head, in one pass (differentiable).
PagedKVCache, paged_attention(q, k_pages, v_pages, page_table, kv_lens, ...)
    A paged cache of keys and values (reserve, write, append, fork, free, compact) and the
    attention of new tokens over it, from one token a sequence to long chunks.
shared_prefix(page_table, kv_lens, cu_seqlens_q, cu_groups, page_size)
    The plan with which that attention reads what forked sequences share once for all.
token_logprobs(logits, targets, top=0)
    Log probabilities of given tokens and the entropy (both differentiable), and the
    likeliest alternatives.
RingHealth, PeerLostError
    Liveness gate for ring calls (`ring_attention(..., health=RingHealth())`).
RingAttentionBlock, RingTransformerLM, shard_targets
    Model layer whose attention is the ring (models/).
"""
from .version import __version__  # noqa: F401
from .parallel.layouts import RingLayout, make_layout  # noqa: F401
from .parallel.api import ring_attention  # noqa: F401
from .parallel.health import PeerLostError, RingHealth  # noqa: F401
from .ops.flash import KernelStatusError, flash_attn, flash_attn_bwd, flash_attn_fwd  # noqa: F401
from .ops.logprobs import TokenLogprobs, token_logprobs  # noqa: F401
from .ops.norm import rms_norm, rms_norm_fp8  # noqa: F401
from .ops.paged import PagedKVCache, SharedPrefix, paged_attention, shared_prefix  # noqa: F401
from .ops.rotary import apply_norm_rotary, apply_rotary, rotary_frequencies  # noqa: F401
from .ops.graphs import GraphedAttention  # noqa: F401
from .models import RingAttentionBlock, RingTransformerLM, shard_targets  # noqa: F401
