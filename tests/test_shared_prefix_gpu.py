"""Attention of sequences that share a prefix against plain attention of each in 64 bits
(test_paged_attention_gpu.py's, whose tolerances hold: joining fp32 parts adds a few steps of
2^-24, which its 4e-5 of the weights contains), and shared_prefix()'s plan against the page
table."""
import pytest
import torch

from test_paged_attention_gpu import Problem

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Forked(Problem):
    """Groups of (prefix, [(own tokens, new tokens), ...]): each group's sequences hold the same
    pages for the prefix's full ones; the rest of it is copied into pages of their own."""

    def __init__(self, groups, heads, kv_heads, D, page, dtype=torch.bfloat16, seed=0, tail=0, big=1.0):
        new = [n for _, members in groups for _, n in members]
        kv = [prefix + own for prefix, members in groups for own, _ in members]
        super().__init__(new, kv, heads, kv_heads, D, page, dtype, seed, tail=tail, big=big)
        self.cg, b = [0], 0
        table = self.table.tolist()
        for prefix, members in groups:
            lead, full = b, prefix // page
            for i in range(len(members)):
                if i:
                    for j in range(full):  # the pages are the first one's; those it had become NaN
                        old = table[b][j]
                        self.k[old] = self.v[old] = float("nan")
                        table[b][j] = table[lead][j]
                    for mine, first, pool in ((self.keys, self.keys[lead], self.k), (self.values, self.values[lead], self.v)):
                        mine[b][:prefix] = first[:prefix]
                        for t in range(full * page, prefix):
                            pool[table[b][t // page], t % page] = first[t]
                b += 1
            self.cg.append(b)
        self.table = _ints(table)
        self.groups = _ints(self.cg)

    def plan(self, **kw):
        from multi_gpu_flashattention_b200 import shared_prefix
        return shared_prefix(self.table, self.lens, self.cu, kw.pop("groups", self.groups), self.page, **kw)

    def both(self, least=None, **kw):
        plan = self.plan()
        want = self.expected(self.cg)
        assert plan.lens.tolist() == want
        if least is not None:
            assert max(want) >= least
        for causal in (True, False):
            out, lse = self.run(causal=causal, shared=plan, **kw)
            self.check(out, lse, causal)
        return plan

    def expected(self, cg):
        """The plan, page by page."""
        table, out = self.table.tolist(), []
        for a, e in zip(cg, cg[1:]):
            pages = 0
            if e - a > 1:
                most = min((self.kv[b] - self.new[b]) // self.page for b in range(a, e))
                while pages < most and len({table[b][pages] for b in range(a, e)}) == 1:
                    pages += 1
            out.append(pages * self.page)
        return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,D,page", [(4, 4, 64, 16), (8, 2, 128, 16), (7, 1, 128, 64), (32, 8, 128, 32),
                                                   (16, 1, 64, 128), (32, 1, 128, 16), (48, 1, 64, 16)])
def test_one_token_each(heads, kv_heads, D, page, dtype):
    """Groups of one and of several sequences, prefixes of less than a page, of full pages, of
    pages and a part; own tokens from the new one alone on."""
    groups = [(500, [(1, 1), (2, 1), (33, 1), (400, 1)]), (page - 1, [(1, 1), (70, 1)]), (300, [(5, 1)]),
              (4 * page, [(1, 1)] * 3), (1, [(1, 1), (1, 1)])]
    Forked(groups, heads, kv_heads, D, page, dtype).both(least=256)


@pytest.mark.parametrize("members", [2, 8, 16, 17, 33, 70, 129, 300])
def test_group_sizes(members):
    """From rows that the decode kernel takes, to several units of 256 rows."""
    g = torch.Generator().manual_seed(members)
    own = torch.randint(1, 60, (members,), generator=g).tolist()
    Forked([(700, [(n, 1) for n in own])], 8, 2, 128, 16, seed=members).both(least=600)


def test_large_and_small_groups_in_one_call():
    groups = [(900, [(7, 1)] * 40), (333, [(90, 1), (3, 1)]), (20, [(4, 1)] * 5), (2000, [(1, 1)] * 20), (64, [(200, 1)])]
    Forked(groups, 16, 4, 64, 32, tail=9).both()


@pytest.mark.parametrize("new", [2, 4, 8, 9, 40, 300])
def test_several_new_tokens(new):
    """Speculative tokens and chunks, in both kernels, of which a sequence may have fewer or none."""
    groups = [(640, [(new, new), (new + 30, new), (new + 1, 1), (5, 0)]), (100, [(new, new - 1), (new + 77, new)]),
              (50, [(new, new)])]
    Forked(groups, 8, 2, 128, 16, seed=new).both()


@pytest.mark.parametrize("prefix,members", [(30000, 4), (9000, 40)])
def test_long_prefix(prefix, members):
    Forked([(prefix, [(3 + i, 1) for i in range(members)])], 8, 2, 128, 64).both(least=8000)


def test_large_scores():
    Forked([(500, [(20, 1)] * 5), (500, [(20, 1)] * 40)], 8, 2, 64, 16, torch.float16, big=4.0).both()


def test_rows_outside_and_strides():
    """Rows of no sequence keep what they held; q and out are cut from wider tensors; slots in
    any order."""
    from multi_gpu_flashattention_b200 import paged_attention, shared_prefix
    p = Forked([(200, [(5, 1)] * 3), (90, [(9, 2), (4, 2)])], 8, 2, 64, 16, tail=6)
    T = p.q.shape[0]
    wide = torch.randn(T, 12, 64, device="cuda", dtype=p.dtype)
    wide[:, 2:10] = p.q
    out = torch.full((T, 20, 64), 5.0, device="cuda", dtype=p.dtype)
    order = [3, 0, 4, 1, 2]
    slots = _ints([order.index(b) for b in range(5)])
    table, lens = p.table[order].contiguous(), p.lens[order].contiguous()
    plan = shared_prefix(table, lens, p.cu, p.groups, 16, slots=slots)
    assert plan.lens.tolist() == p.expected(p.cg)
    o, lse = paged_attention(wide[:, 2:10], p.k, p.v, table, lens, p.cu, 2, slots=slots, out=out[:, 3:11],
                             return_lse=True, shared=plan)
    p.check(o, lse)
    assert (out[-6:] == 5).all() and (out[:, :3] == 5).all() and (out[:, 11:] == 5).all()


def test_plan_follows_the_pages_not_the_groups():
    """Sequences that share nothing, or part; a group that mixes two prompts; sequences of no
    group; new tokens that lie in shared pages."""
    p = Forked([(256, [(5, 1), (6, 1)]), (256, [(5, 1), (6, 1)]), (64, [(16, 1), (16, 1)])], 4, 2, 64, 16)
    for cg in ([0, 4, 6], [0, 2, 6], [1, 3, 5], [2, 4], [0, 0, 2, 2, 6, 6], [6], [3, 3]):
        plan = p.plan(groups=_ints(cg))
        assert plan.lens.tolist() == p.expected(cg)
        first, member = plan.plan[len(cg) - 1:].view(2, 6).tolist()
        for b in range(6):
            g = [i for i, (a, e) in enumerate(zip(cg, cg[1:])) if a <= b < e]
            assert member[b] == (g[0] if g else -1) or len(cg) == 1
            assert first[b] == (plan.lens.tolist()[g[0]] if g else 0) or len(cg) == 1
        p.check(*p.run(shared=plan))
    # both copies end inside the shared pages, with their last 20 tokens new
    q = Forked([(128, [(1, 1), (1, 1)])], 4, 2, 64, 16)
    q.kv = [100, 128]
    q.lens = _ints(q.kv)
    q.new = [20, 20]
    q.cu, q.max_new = _ints([0, 20, 40]), 20
    q.q = torch.randn(40, 4, 64, device="cuda").bfloat16()
    q.keys, q.values = [[t[:n] for t, n in zip(x, q.kv)] for x in (q.keys, q.values)]
    plan = q.plan()
    assert plan.lens.tolist() == [80]
    q.check(*q.run(shared=plan))


def test_same_bits_again_and_beside_other_work():
    p = Forked([(3000, [(9, 1)] * 12), (3000, [(9, 1)] * 60)], 16, 4, 128, 64)
    plan = p.plan()
    first = p.run(shared=plan)
    for _ in range(5):
        p.run()
        again = p.run(shared=p.plan())
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_captured_with_lengths_that_grow():
    p = Forked([(600, [(200, 1)] * 30)], 8, 2, 64, 16)
    lens = p.lens.clone()
    p.lens.fill_(605)

    def step():
        return p.run(shared=p.plan())

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for kv in (601, 640, 700, int(lens[0])):
        p.lens.fill_(kv)
        graph.replay()
        p.kv = [kv] * 30
        q = p.keys, p.values
        p.keys, p.values = [t[:kv] for t in p.keys], [t[:kv] for t in p.values]
        p.check(out, lse)
        p.keys, p.values = q


def test_cache_forks_and_streams():
    """reserve, append, fork and attend with what the forks share, on a side stream."""
    from multi_gpu_flashattention_b200 import PagedKVCache, rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache = PagedKVCache.allocate(2, 200, 16, 2, 64, 12, 600)
        g = torch.Generator("cuda").manual_seed(0)
        make = lambda n, h: torch.randn(n, h, 64, device="cuda", generator=g).bfloat16()
        pos = cache.reserve([0], [0, 150], 150)
        for layer in range(2):
            cache.append(layer, make(150, 4), make(150, 2), make(150, 2), pos, inv, [0], [0, 150])
        cache.fork([0] * 7, list(range(1, 8)))
        slots, cu = list(range(8)), list(range(9))
        for _ in range(20):
            pos = cache.reserve(slots, cu, 8)
            shared = cache.shared_prefix(slots, cu, [0, 8])
            for layer in range(2):
                q = cache.append(layer, make(8, 4), make(8, 2), make(8, 2), pos, inv, slots, cu)
                a, la = cache.attend(layer, q, slots, cu, 1, return_lse=True, shared=shared)
                b, lb = cache.attend(layer, q, slots, cu, 1, return_lse=True)
                # both within u |out| + (u + 4e-5) mean |v| of the same, u = 2^-9 + ...
                u = 2.0 ** -8
                assert ((a.float() - b.float()).abs() <= 2 * (u * b.float().abs() + (u + 4e-5) * 4.5)).all()
                assert ((la - lb).abs() <= 4e-5 * (1 + lb.abs())).all()
        assert shared.lens.tolist() == [144]
    side.synchronize()


def test_refusals_and_errors_on_the_device():
    from multi_gpu_flashattention_b200 import KernelStatusError, SharedPrefix, shared_prefix
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    p = Forked([(100, [(5, 1), (6, 1)])], 4, 2, 64, 16)
    plan = p.plan()
    for match, kw in (("cu_groups must be", dict(groups=p.groups.long())), ("cu_groups must be", dict(groups=p.groups.cpu())),
                      ("cu_groups must be", dict(groups=p.groups[:0]))):
        with pytest.raises(RuntimeError, match=match):
            p.plan(**kw)
    with pytest.raises(RuntimeError, match="page size must be"):
        shared_prefix(p.table, p.lens, p.cu, p.groups, 24)
    with pytest.raises(RuntimeError, match="of another batch"):
        p.run(shared=SharedPrefix(p.groups, plan.plan[:-1].clone()))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        shared_prefix(p.table.cpu(), p.lens.cpu(), p.cu.cpu(), p.groups.cpu(), 16)
    # groups that fall or leave the batch: an error, nothing shared, the answers right
    for cg in ([0, 3], [2, 0], [-1, 2], [0, 2, 1, 2]):
        bad = p.plan(groups=_ints(cg))
        assert not any(bad.lens.tolist())
        with pytest.raises(KernelStatusError):
            check_errors()
        out, lse = p.run(shared=bad)
        torch.cuda.synchronize()
        p.check(out, lse)
        try:
            check_errors()  # the attention may report the groups again
        except KernelStatusError:
            pass
    # a plan whose lengths do not fit the batch is reported, and reads nothing outside
    for lens in ([96 + 16 * 1000] * 3, [7] * 3, [-16] * 3):
        wrong = SharedPrefix(p.groups, _ints(lens + [0, 0]))
        p.run(shared=wrong)
        with pytest.raises(KernelStatusError):
            check_errors()


@pytest.mark.parametrize("heads,kv_heads", [(64, 1), (128, 1), (128, 2), (66, 2)])
@pytest.mark.parametrize("new", [1, 3])
def test_many_heads_a_key_head(heads, kv_heads, new):
    Forked([(300, [(20, new)] * 3), (90, [(7, new)]), (70, [(40, new)] * 2)], heads, kv_heads, 64, 16).both(least=288)


def test_members_without_new_tokens():
    """Also at a group's head and end, and groups of nothing else."""
    Forked([(200, [(9, 0), (9, 1), (40, 2), (8, 0)]), (100, [(3, 0), (4, 0)]), (64, [(5, 1)] * 2)], 8, 2, 128, 16).both(least=192)


def test_a_row_named_twice():
    """Two sequences of a batch that read one row of the table: as without the plan."""
    from multi_gpu_flashattention_b200 import shared_prefix
    p = Forked([(500, [(20, 1), (31, 1)])], 8, 2, 64, 16)
    slots, groups = _ints([1, 1]), _ints([0, 2])
    plan = shared_prefix(p.table, p.lens, p.cu, groups, p.page, slots=slots)
    assert plan.lens.tolist() == [(531 - 1) // 16 * 16]
    args = (p.q, p.k, p.v, p.table, p.lens, p.cu, 1)
    from multi_gpu_flashattention_b200 import paged_attention
    a, la = paged_attention(*args, slots=slots, return_lse=True, shared=plan)
    b, lb = paged_attention(*args, slots=slots, return_lse=True)
    # each within u |out| + (u + 4e-5) max |v| of the same value
    u, most = 2.0 ** -8, max(float(v.abs().max()) for v in p.values)
    assert ((a.float() - b.float()).abs() <= 2 * (u * b.float().abs() + (u + 4e-5) * most)).all()
    assert ((la - lb).abs() <= 4e-5 * (1 + lb.abs())).all()


def test_two_streams_and_two_graphs():
    """Calls under way side by side, and captured ones replayed in turn and side by side, have
    workspaces of their own: the bits are those of a call alone."""
    ps = [Forked([(3000, [(9, 1)] * 12), (2000, [(300, 1)] * 40)], 16, 4, 128, 64, seed=1),
          Forked([(700, [(200, 1)] * 30)], 8, 2, 64, 16, seed=2)]
    alone = [p.run(shared=p.plan()) for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for p, s in zip(ps, streams):
            with torch.cuda.stream(s):
                got.append(p.run(shared=p.plan()))
        torch.cuda.synchronize()
        for x, y in zip(alone, got):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
    graphs = []
    for p in ps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = p.run(shared=p.plan())
        graphs.append((g, out))
    for side in (False, True):
        for _ in range(5):
            for (g, out), s in zip(graphs, streams):
                for t in out:
                    t.zero_()
            torch.cuda.synchronize()
            for (g, out), s in zip(graphs, streams):
                with torch.cuda.stream(s if side else torch.cuda.current_stream()):
                    g.replay()
            torch.cuda.synchronize()
            for x, (g, out) in zip(alone, graphs):
                assert torch.equal(x[0], out[0]) and torch.equal(x[1], out[1])
