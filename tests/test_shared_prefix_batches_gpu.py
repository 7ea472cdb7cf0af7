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
