"""A paged cache of keys and values on the device, and attention over it.

The cache's memory is a pool of pages, each `page_size` tokens of one sequence; a
sequence is a slot, whose row of the page table names its pages in order. Every step
runs on the device: the host need not know a length, nothing synchronises, and each
call can be captured into a CUDA graph.

    cache = PagedKVCache.allocate(n_layers, pages, page_size, kv_heads, head_dim, ...)
    pos = cache.reserve(slots, cu_seqlens, n_tokens)        # room for a batch of new tokens
    for layer ...:
        q, k = apply_rotary(q, k, pos, inv_freq)
        cache.write(layer, k, v, slots, cu_seqlens)
        out = cache.attend(layer, q, slots, cu_seqlens, max_seqlen_q)
    cache.fork(src, dst); cache.free(slots); cache.compact()

append() does the rotary positions, head norms and the write in one pass; sequences forked
from one prompt, a group's one behind another in the batch, read it once:

    shared = cache.shared_prefix(slots, cu_seqlens, cu_groups)   # once a step
    for layer ...:
        q = cache.append(layer, q, k, v, pos, inv_freq, slots, cu_seqlens)
        out = cache.attend(layer, q, slots, cu_seqlens, max_seqlen_q, shared=shared)

A batch packs its sequences' new tokens: sequence b's are the rows
[cu_seqlens[b], cu_seqlens[b + 1]). Rows outside every sequence (a batch padded for a
graph) are left alone: outputs keep what they held there.

What goes wrong on the device (a slot out of range or named twice, a row of the page
table that is too short, too few free pages, a page that is not in the pool) leaves the
sequence concerned as it was and faults nothing; the batch's other sequences are served.
It raises KernelStatusError at a later call on the device, of this or another cache, or
in check_errors(): reserve() raises before it changes anything, so the call can be made
again; free(), fork() and compact() raise after they have done their own work; so do, before
theirs, token_logprobs() and the functions paged_attention() and shared_prefix() without a
status of their own; write(), append(), shared_prefix() and attend() of a cache, in the
middle of a step, do not raise it. A slot that a batch names twice
is the first naming's. A cache has less than 2^30 pages and 2^31 page table entries, a batch less
than 2^30 rows.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Union

import torch

from .._ext import C
from .flash import DEFAULT_WAIT_LIMIT_NS, host_status

Ints = Union[torch.Tensor, Sequence[int]]


def _scale(head_dim: int, softmax_scale: Optional[float]) -> float:
    return softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(head_dim)


class SharedPrefix(NamedTuple):
    """What the sequences of a batch share (shared_prefix()): cu_groups, the groups; plan, int32,
    the tokens that each group shares, then each sequence's, then its group (below 0: it shares
    nothing)."""
    cu_groups: torch.Tensor
    plan: torch.Tensor

    @property
    def lens(self) -> torch.Tensor:
        """int32 [groups]: how many tokens each group shares."""
        return self.plan[:self.cu_groups.shape[0] - 1]


def _status_word(device, status: Optional[torch.Tensor]) -> torch.Tensor:
    if status is not None:
        return status
    h = host_status(device)
    h.poll()  # an error of an earlier call surfaces here
    return h.word


def shared_prefix(page_table: torch.Tensor, kv_lens: torch.Tensor, cu_seqlens_q: torch.Tensor,
                  cu_groups: torch.Tensor, page_size: int, slots: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None) -> SharedPrefix:
    """The plan with which paged_attention reads what sequences share once for all of them.

    cu_groups int32 [groups + 1]: group g is the batch's sequences [cu_groups[g],
    cu_groups[g + 1]), neighbours, as forks of one prompt. Those with new tokens share the
    leading pages that the page table names alike for all of them, as far as these are full
    and hold none of their new tokens; one alone, or outside every group, shares nothing. A
    group may keep sequences that have ended: without new tokens they change nothing,
    whether they are freed or not. The other
    arguments are those of paged_attention, whose batch the plan is of: it holds until the
    lengths or the page table change, hence for all layers of a step. Up to 4096 sequences
    and groups. Everything stays on the device. cu_groups that fall or leave the batch are
    reported as an error, and nothing is shared.

    It pays for sequences of one new token each where much need not be read again: (members
    - 1) times the prefix's keys and values, in one layer, of 0.25 to 0.5 GB and more (on one
    B200 1.2 to 12 times as fast as without). Below that, and mostly for several new tokens
    and for chunks, paged_attention without a plan is faster (by up to 2 to 4 times where
    little is shared): it is one launch or two, and finds a short prefix in L2."""
    plan = C().shared_prefix(page_table, kv_lens, cu_seqlens_q, cu_groups, page_size, slots,
                             _status_word(page_table.device, status))
    return SharedPrefix(cu_groups, plan)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, kv_lens: torch.Tensor, cu_seqlens_q: torch.Tensor,
                    max_seqlen_q: int, slots: Optional[torch.Tensor] = None, causal: bool = True,
                    softmax_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    return_lse: bool = False, status: Optional[torch.Tensor] = None,
                    wait_limit_ns: int = DEFAULT_WAIT_LIMIT_NS, shared: Optional[SharedPrefix] = None):
    """Attention of each sequence's new tokens over its paged keys and values.

    q [tokens, heads, D] (bfloat16 or float16, D = 64 or 128), the sequences' new tokens
    one behind another: sequence b's are rows [cu_seqlens_q[b], cu_seqlens_q[b + 1]), at
    most max_seqlen_q. k_pages, v_pages [pages, page_size, kv_heads, D] of q's dtype,
    page_size a power of two from 16 to 1024, heads a multiple of kv_heads (up to 128
    times). page_table int32 [rows, width] names each sequence's pages, kv_lens int32
    [rows] its tokens, the new ones included; `slots` int32 [sequences] gives the row of
    each sequence (default: row b). Up to 4096 sequences; the int32 tensors contiguous.
    max_seqlen_q also decides between the kernels for few and for many rows. shared: the
    batch's shared_prefix(), with which keys and values that sequences share are read once
    (when that pays, it says); such a call takes a workspace of 8 * tokens * heads * (D + 2)
    bytes.

    The new tokens are the sequence's last: token i of n sees keys [0, kv_len - n + i],
    or with causal=False all kv_len. A token that sees no key gets 0, and -inf for its
    LSE. Keys and values behind kv_len are never used, whatever they hold; values at
    places that only some of a sequence's new tokens see have to be finite.
    Returns out (q's dtype and shape, into `out` if given) or, with return_lse, (out,
    fp32 natural-log LSE [heads, tokens]). Rows of q outside every sequence are not
    written. Inference only: there is no gradient."""
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
        raise RuntimeError("paged_attention has no gradient: call it under torch.no_grad()")
    status = _status_word(q.device, status)
    o, lse = C().paged_attention(q, k_pages, v_pages, page_table, kv_lens, cu_seqlens_q,
                                 max_seqlen_q, slots, causal, _scale(q.shape[-1], softmax_scale),
                                 out, return_lse, status, wait_limit_ns, *(shared or (None, None)))
    return (o, lse) if return_lse else o


class PagedKVCache:
    """Keys and values of up to `slots` sequences in a pool of pages shared by all layers.

    k, v        [layers, pages, page_size, kv_heads, D], bfloat16 or float16, D 64 or 128
    page_table  int32 [slots, width]: a sequence's pages in order, -1 behind them
    lens        int32 [slots]: its tokens
    refs        int32 [pages]: how many sequences hold the page; 0: it is free
    grown       int32 [slots]: the tokens that the last reserve() added (0: none or not
                enough pages), which write() fills

    The tensors are the caller's (allocate() makes them); all are contiguous but k and v,
    whose outer dimensions may be strided. Pages are always taken lowest first, in the
    order of a call's sequences, so results do not depend on timing. Calls on one cache
    have to be ordered by the caller where they run on several streams. Slots are int32
    CUDA tensors, or sequences of numbers, which are copied."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
                 lens: torch.Tensor, refs: torch.Tensor, grown: torch.Tensor):
        C().cache_check(k, v, page_table, lens, refs, grown)
        self.k, self.v, self.page_table = k, v, page_table
        self.lens, self.refs, self.grown = lens, refs, grown
        self.page_size = k.shape[2]
        self._layers = list(zip(k.unbind(0), v.unbind(0)))
        self._status = host_status(k.device)
        self._state = (page_table, lens, refs, grown, self._status.word)

    @classmethod
    def allocate(cls, n_layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 slots: int, max_tokens: int, dtype=torch.bfloat16, device="cuda") -> "PagedKVCache":
        """An empty cache; a sequence may grow to max_tokens."""
        device = torch.empty(0, device=device).device
        shape = (n_layers, pages, page_size, kv_heads, head_dim)
        ints = dict(dtype=torch.int32, device=device)
        k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        return cls(k, v, torch.full((slots, -(-max_tokens // page_size)), -1, **ints),
                   torch.zeros(slots, **ints), torch.zeros(pages, **ints), torch.zeros(slots, **ints))

    def _ints(self, x: Ints) -> torch.Tensor:
        return x if isinstance(x, torch.Tensor) else torch.tensor(x, dtype=torch.int32, device=self.k.device)

    def reserve(self, slots: Ints, cu_seqlens: Ints, n_tokens: int) -> torch.Tensor:
        """Room for the batch's new tokens: sequence slots[b] grows by cu_seqlens[b + 1] -
        cu_seqlens[b] tokens, and gets pages for them. Returns the new tokens' positions,
        int32 [n_tokens] (0 for rows outside every sequence). A sequence that cannot get
        all its pages does not grow: refused() tells its rows."""
        self._status.poll()
        return C().cache_reserve(self.k, *self._state, self._ints(slots), self._ints(cu_seqlens), n_tokens)

    def refused(self, slots: Ints, cu_seqlens: Ints, n_tokens: int) -> torch.Tensor:
        """Which rows of the batch belong to a sequence that reserve(), called with the same
        arguments just before, left as it was: bool [n_tokens], on the device. What attend()
        returns for these rows stands for nothing."""
        return C().cache_refused(self.k, *self._state, self._ints(slots), self._ints(cu_seqlens), n_tokens)

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: Ints, cu_seqlens: Ints) -> None:
        """The keys and values [tokens, kv_heads, D] of the batch that reserve() made room
        for, with the same slots and cu_seqlens."""
        C().cache_write(self.k, self.v, *self._state, layer, k, v, self._ints(slots), self._ints(cu_seqlens))

    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               positions: torch.Tensor, inv_freq: torch.Tensor, slots: Ints, cu_seqlens: Ints,
               q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
               eps: float = 1e-6, interleaved: bool = False, magnitude: float = 1.0) -> torch.Tensor:
        """write() with the rotary positions applied on the way, in one pass: q [tokens,
        heads, D] and k [tokens, kv_heads, D] become what apply_rotary or, with weights,
        apply_norm_rotary makes of them; k's and v go to the pages of the batch that
        reserve() made room for, and q's are returned (of all rows). positions int32 or int64
        [tokens], as reserve() returns them; the rest as in those functions. Inference only:
        there is no gradient."""
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, q_weight, k_weight)):
            raise RuntimeError("append has no gradient: call it under torch.no_grad()")
        return C().cache_append(self.k, self.v, *self._state, layer, q, k, v, positions, inv_freq,
                                self._ints(slots), self._ints(cu_seqlens), q_weight, k_weight, eps,
                                interleaved, magnitude)

    def attend(self, layer: int, q: torch.Tensor, slots: Ints, cu_seqlens: Ints, max_seqlen_q: int,
               causal: bool = True, softmax_scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False,
               shared: Optional[SharedPrefix] = None):
        """paged_attention of the batch's queries [tokens, heads, D] over a layer's cache;
        shared: the batch's shared_prefix()."""
        if not 0 <= layer < len(self._layers):
            raise IndexError(f"layer {layer} is not one of the cache's {len(self._layers)}")
        k, v = self._layers[layer]
        return paged_attention(q, k, v, self.page_table, self.lens, self._ints(cu_seqlens),
                               max_seqlen_q, slots=self._ints(slots), causal=causal,
                               softmax_scale=softmax_scale, out=out, return_lse=return_lse,
                               status=self._status.word, shared=shared)

    def shared_prefix(self, slots: Ints, cu_seqlens: Ints, cu_groups: Ints) -> SharedPrefix:
        """shared_prefix() of a batch that reserve() has made room for: cu_groups [groups + 1]
        says which of its sequences, neighbours, were forked from one another. For attend()
        in every layer of the step."""
        return shared_prefix(self.page_table, self.lens, self._ints(cu_seqlens), self._ints(cu_groups),
                             self.page_size, slots=self._ints(slots), status=self._status.word)

    def fork(self, src: Ints, dst: Ints, share: bool = True) -> None:
        """Sequence dst[i] becomes a copy of src[i]. Full pages are held by both, and the
        tokens of a last page that is not full are copied to a page of dst's own, in all
        layers; share=False copies every page. dst has to be empty, and none of the
        call's sources; a source may be forked several times. Tokens that are reserved but
        not yet written in a layer are copied as they are: fork before reserve(), or after
        the last layer's write()."""
        C().cache_fork(self.k, self.v, *self._state, self._ints(src), self._ints(dst), share)
        self._status.poll()

    def free(self, slots: Ints) -> None:
        """Empties the sequences; pages that no other holds become free."""
        C().cache_free(self.k, *self._state, self._ints(slots))
        self._status.poll()

    def compact(self) -> None:
        """Moves the pages in use to the front of the pool, in all layers, and changes the
        page table to match; the free pages are the last ones then."""
        C().cache_compact(self.k, self.v, *self._state)
        self._status.poll()

    def free_pages(self) -> int:
        """How many pages are free (waits for the device)."""
        return int((self.refs == 0).sum())
