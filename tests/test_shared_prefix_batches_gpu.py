"""Batches over shared prefixes that take several launches: what is wrong with a sequence is
reported as without the plan, and faults nothing."""
import pytest
import torch

from test_shared_prefix_gpu import Forked, _ints

pytestmark = pytest.mark.gpu


def _batch(kv_heads=2, group=4, new=None, **kw):
    """38 sequences, one token each but as `new` says (a dict): a group of 28, whose rows fill
    128-row tiles, one of 6, and 4 of no group. With the sequences' own keys three launches."""
    new = new or {}
    n = lambda b: new.get(b, 1)
    groups = [(200, [(3 + b, n(b)) for b in range(28)]), (120, [(5 + b, n(b)) for b in range(28, 34)]),
              *((90, [(7, n(b))]) for b in range(34, 38))]
    p = Forked(groups, kv_heads * group, kv_heads, 64, 16, **kw)
    p.groups = _ints([0, 28, 34])
    return p


@pytest.mark.parametrize("kv_heads", [2, 4])  # a key head's units, and four heads' at once
@pytest.mark.parametrize("b", [0, 9, 27, 28, 33, 36])
def test_wrong_contents_are_reported(b, kv_heads):
    """Slots out of range, lengths below 0 and beyond the table: an error word, no fault, and the
    other sequences are right."""
    from multi_gpu_flashattention_b200 import KernelStatusError
    from multi_gpu_flashattention_b200.ops.flash import check_errors

    def wrong(change):
        p = _batch(kv_heads)
        slots = _ints(list(range(38)))
        change(p, slots)
        out, lse = p.run(slots=slots, shared=p.plan(slots=slots))
        with pytest.raises(KernelStatusError):
            check_errors()
        check_errors()  # re-armed
        p.new[b] = 0  # (its rows stand for nothing)
        p.check(out, lse)

    check_errors()
    wrong(lambda p, s: s.__setitem__(b, 38))
    wrong(lambda p, s: s.__setitem__(b, -1))
    wrong(lambda p, s: p.lens.__setitem__(b, -5))
    wrong(lambda p, s: p.lens.__setitem__(b, 1 << 30))


@pytest.mark.parametrize("kv_heads", [2, 4])
@pytest.mark.parametrize("b", [0, 27, 30, 36])
def test_more_tokens_than_announced_are_reported(b, kv_heads):
    from multi_gpu_flashattention_b200 import KernelStatusError
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    p = _batch(kv_heads, new={b: 2})
    out = torch.full_like(p.q, 5.0)
    check_errors()
    _, lse = p.run(out=out, max_new=1, shared=p.plan())
    with pytest.raises(KernelStatusError):
        check_errors()
    assert (out[b:b + 2] == 5.0).all()
    p.new[b] = 0
    p.check(out, lse)


@pytest.mark.parametrize("b", [0, 9, 27, 30])
def test_a_plan_of_longer_sequences_is_reported(b):
    """A sequence that has become shorter than what the plan says it shares."""
    from multi_gpu_flashattention_b200 import KernelStatusError
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    p = _batch()
    plan = p.plan()
    p.lens[b] = 50
    check_errors()
    out, lse = p.run(shared=plan)
    with pytest.raises(KernelStatusError):
        check_errors()
    p.new[b] = 0
    p.check(out, lse)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("groups,heads,kv_heads", [(64, 4, 2), (1, 4, 4)])
def test_as_many_sequences_and_groups_as_a_call_takes(groups, heads, kv_heads, D):
    """4096 in all: the kernels' tables of them take the most shared memory."""
    per = (4096 - groups) // groups
    sizes = [per] * (groups - 1) + [4096 - groups - per * (groups - 1)]
    p = Forked([(16 + 16 * (g % 3), [(1 + i % 5, 1) for i in range(n)]) for g, n in enumerate(sizes)],
               heads, kv_heads, D, 16)
    plan = p.plan()
    assert plan.lens.tolist() == p.expected(p.cg)
    p.check(*p.run(shared=plan))
    with pytest.raises(RuntimeError, match="at most 4096 sequences and groups"):
        p.plan(groups=_ints(p.cg + [p.cg[-1]]))


@pytest.mark.parametrize("gone", [[0], [5], [0, 1, 2], [27], [3, 9, 20], list(range(27)), list(range(28))])
def test_sequences_that_have_ended_end_no_sharing(gone):
    """Freed members without new tokens, first ones too; one that is left alone shares nothing."""
    p = _batch(new={b: 0 for b in gone})
    for b in gone:
        p.table[b] = -1
        p.lens[b] = 0
    plan = p.plan()
    left = 28 - len(gone)
    assert plan.lens.tolist() == [192 if left > 1 else 0, 112]
    first, member = plan.plan[2:].view(2, 38).tolist()
    for b in range(28):
        assert first[b] == (0 if b in gone or left == 1 else 192)
        assert (member[b] == 0) == (b not in gone)
    for causal in (True, False):
        p.check(*p.run(causal=causal, shared=plan), causal)


def test_a_slot_out_of_range_ends_no_sharing():
    """Of the first of a group, with a new token: an error, and the others share as before."""
    from multi_gpu_flashattention_b200 import KernelStatusError
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    p = _batch()
    slots = _ints(list(range(38)))
    slots[0] = slots[29] = 38
    plan = p.plan(slots=slots)
    assert plan.lens.tolist() == [192, 112]
    out, lse = p.run(slots=slots, shared=plan)
    with pytest.raises(KernelStatusError):
        check_errors()
    p.new[0] = p.new[29] = 0
    p.check(out, lse)


def test_a_captured_batch_whose_answers_end_one_by_one():
    """A padded batch of a fixed form, whose sequences are freed between replays: the rest share
    the prompt's pages to the last pair."""
    from multi_gpu_flashattention_b200 import PagedKVCache
    g = torch.Generator("cuda").manual_seed(0)
    make = lambda n, h: torch.randn(n, h, 64, device="cuda", generator=g).bfloat16()
    cache = PagedKVCache.allocate(1, 200, 16, 2, 64, 12, 600)
    cache.reserve([0], [0, 150], 150)
    cache.write(0, make(150, 2), make(150, 2), [0], [0, 150])
    cache.fork([0] * 11, list(range(1, 12)))
    slots, cu, groups = _ints(list(range(12))), _ints(list(range(13))), _ints([0, 12])
    k, v, q = make(12, 2), make(12, 2), make(12, 4)
    a, b = torch.zeros_like(q), torch.zeros_like(q)

    def step():
        cache.reserve(slots, cu, 12)
        shared = cache.shared_prefix(slots, cu, groups)
        cache.write(0, k, v, slots, cu)
        cache.attend(0, q, slots, cu, 1, out=a, shared=shared)
        cache.attend(0, q, slots, cu, 1, out=b)
        return shared.lens

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens = step()
    live = list(range(12))
    for end in (0, 7, 1, 11, 4, 2, 3, 10, 5, 6):
        live.remove(end)
        cache.free([end])
        # the rows stay packed, the ended sequences take none
        cu.copy_(_ints([sum(s in live for s in range(i)) for i in range(13)]))
        graph.replay()
        assert lens.tolist() == [144]
        n, u = len(live), 2.0 ** -8
        # (as in test_cache_forks_and_streams)
        x, y = a[:n].float(), b[:n].float()
        assert ((x - y).abs() <= 2 * (u * y.abs() + (u + 4e-5) * 4.5)).all()


@pytest.mark.parametrize("small", [False, True])
@pytest.mark.parametrize("first,last", [(-1, 0), (0, 1), (-2, 3)])
def test_rows_that_leave_the_batch_are_reported(first, last, small):
    """cu_seqlens that begins below 0 and ends behind the tokens: the sequences there are not
    served, the others of their groups are, with their prefix; in three launches and in one."""
    from multi_gpu_flashattention_b200 import KernelStatusError
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    p = Forked([(200, [(9, 1)] * 4)] if small else [(200, [(9, 1)] * 28), (120, [(9, 1)] * 10)], 8, 2, 64, 16)
    n = len(p.kv)
    p.cu[0] += first
    p.cu[n] += last
    plan = p.plan()
    assert plan.lens.tolist() == ([192] if small else [192, 112])
    check_errors()
    out, lse = p.run(max_new=4, shared=plan)
    with pytest.raises(KernelStatusError):
        check_errors()
    if first:
        p.new[0] = 0
    if last:
        p.new[n - 1] = 0
    p.check(out, lse)


def test_half_a_plan_is_refused():
    from multi_gpu_flashattention_b200 import SharedPrefix
    p = Forked([(100, [(5, 1), (6, 1)])], 4, 2, 64, 16)
    for half in (SharedPrefix(p.groups, None), SharedPrefix(None, p.plan().plan)):
        with pytest.raises(RuntimeError, match="come together"):
            p.run(shared=half)
    p.check(*p.run(shared=p.plan()))
