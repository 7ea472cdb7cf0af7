"""PagedKVCache against a cache kept on the host: which pages every sequence holds, the
reference counts, and every token's keys and values. Everything here is copies and whole
numbers, so all comparisons are exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu

H, D = 2, 64


class Model:
    """The same cache in Python: rows of pages, counts, and each sequence's tokens."""

    def __init__(self, pages, page, slots, width):
        self.page, self.width = page, width
        self.refs = [0] * pages
        self.rows = [[] for _ in range(slots)]
        self.lens, self.grown = [0] * slots, [0] * slots
        self.tokens = [[] for _ in range(slots)]  # per sequence: ids of its tokens

    def _lowest(self, n):
        free = [i for i, r in enumerate(self.refs) if r == 0][:n]
        return free if len(free) == n else None

    def reserve(self, slots, new):
        pos, seen, short = [], set(), False
        for s, n in zip(slots, new):
            pos += list(range(self.lens[s], self.lens[s] + n)) if 0 <= s < len(self.lens) else [None] * n
            if not 0 <= s < len(self.lens) or s in seen:
                continue
            seen.add(s)
            self.grown[s] = 0
            want = -(-(self.lens[s] + n) // self.page)
            if want > self.width:
                continue
            need = want - len(self.rows[s])
            if need and (short or self._lowest(need) is None):
                short = True  # the pages are given in order: nobody behind gets one
                continue
            for i in self._lowest(need):
                self.refs[i] = 1
                self.rows[s].append(i)
            self.lens[s] += n
            self.grown[s] = n
        return pos

    def free(self, slots):
        for s in dict.fromkeys(slots):
            for i in self.rows[s]:
                self.refs[i] -= 1
            self.rows[s], self.tokens[s], self.lens[s], self.grown[s] = [], [], 0, 0

    def fork(self, src, dst, share=True):
        short = False
        for a, b in zip(src, dst):
            l = self.lens[a]
            whole = l // self.page if share else 0
            need = len(self.rows[a]) - whole
            if need and (short or self._lowest(need) is None):
                short = True
                continue
            own = self._lowest(need)
            for i in self.rows[a][:whole]:
                self.refs[i] += 1
            for i in own:
                self.refs[i] = 1
            self.rows[b] = self.rows[a][:whole] + own
            self.lens[b], self.grown[b], self.tokens[b] = l, 0, list(self.tokens[a])

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [i for i in range(live) if not self.refs[i]]
        movers = [i for i in range(live, len(self.refs)) if self.refs[i]]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.rows = [[to.get(i, i) for i in r] for r in self.rows]


def _value(ids, layer, what):
    """The key (0) or value (1) of token id in a layer: small whole numbers, exact in 16 bits."""
    base = torch.tensor(ids, device="cuda", dtype=torch.float64)[:, None, None] * 3 + layer * 7 + what * 11
    h = torch.arange(H, device="cuda")[:, None] * 5 + torch.arange(D, device="cuda")[None, :]
    return ((base + h) % 251).to(torch.bfloat16)


class Pair:
    def __init__(self, pages=40, page=16, slots=12, max_tokens=160, layers=2):
        from multi_gpu_flashattention_b200 import PagedKVCache
        self.c = PagedKVCache.allocate(layers, pages, page, H, D, slots, max_tokens)
        self.c.k.fill_(float("nan"))
        self.c.v.fill_(float("nan"))
        self.m = Model(pages, page, slots, self.c.page_table.shape[1])
        self.layers, self.next = layers, 1

    def append(self, slots, new, tail=0):
        total = sum(new)
        cu = [sum(new[:i]) for i in range(len(new) + 1)]
        pos = self.c.reserve(slots, cu, total + tail).tolist()
        want = self.m.reserve(slots, new)
        ids = list(range(self.next, self.next + total))
        self.next += total
        pad = torch.full((tail, H, D), float("nan"), device="cuda", dtype=torch.bfloat16)
        for layer in range(self.layers):
            k, v = (torch.cat([_value(ids, layer, w), pad]) for w in (0, 1))
            self.c.write(layer, k, v, slots, cu)
        seen = set()
        for b, s in enumerate(slots):
            if 0 <= s < len(self.m.lens) and s not in seen:
                seen.add(s)
                if self.m.grown[s] == new[b]:
                    self.m.tokens[s] += ids[cu[b]:cu[b + 1]]
        return pos, want

    def check(self):
        m, c = self.m, self.c
        width = m.width
        assert c.page_table.tolist() == [r + [-1] * (width - len(r)) for r in m.rows]
        assert c.refs.tolist() == m.refs and c.lens.tolist() == m.lens and c.grown.tolist() == m.grown
        for s, ids in enumerate(m.tokens):
            assert len(ids) == m.lens[s]
            if not ids:
                continue
            rows = torch.tensor(m.rows[s], device="cuda")
            for layer in range(self.layers):
                for w, pool in enumerate((c.k, c.v)):
                    got = pool[layer][rows].reshape(-1, H, D)[:len(ids)]
                    assert torch.equal(got, _value(ids, layer, w)), (s, layer, w)


@pytest.fixture(autouse=True)
def _errors_when_asked(monkeypatch):
    """The steps that follow an error run too: it is raised where the test asks for it."""
    from multi_gpu_flashattention_b200.ops.flash import HostStatus
    poll = HostStatus.poll
    monkeypatch.setattr(HostStatus, "poll", lambda self, wait=False: poll(self, wait=True) if wait else None)


def _errors(expected):
    from multi_gpu_flashattention_b200.ops.flash import KernelStatusError, check_errors
    if expected:
        with pytest.raises(KernelStatusError):
            check_errors()
    else:
        check_errors()


@pytest.mark.parametrize("page", [16, 64])
def test_append(page):
    p = Pair(page=page, max_tokens=10 * page)
    for slots, new in (([3, 0, 7], [1, page, page + 1]), ([0, 3], [1, page - 1]), ([7, 0, 3, 1], [0, 2, 1, 5])):
        pos, want = p.append(slots, new, tail=3)
        assert pos == want + [0, 0, 0]
        p.check()
    _errors(False)


def test_many_tokens_at_once():
    """Over 4096 tokens the positions come from a kernel of their own."""
    p = Pair(pages=700, slots=6, max_tokens=6000, layers=1)
    pos, want = p.append([2, 4], [5000, 1777])
    assert pos == want
    p.check()


def test_fork_shares_full_pages_and_copies_the_rest():
    p = Pair()
    p.append([0, 1, 2], [37, 32, 3])
    p.c.fork([0, 0, 1, 2, 5], [6, 7, 8, 9, 10])  # twice the same source; an empty one
    p.m.fork([0, 0, 1, 2, 5], [6, 7, 8, 9, 10])
    p.check()
    p.append([0, 6, 7, 8, 1], [5, 30, 1, 2, 4])  # every branch goes on by itself
    p.check()
    p.c.free([0, 8])
    p.m.free([0, 8])
    p.check()
    p.append([0, 3], [50, 20])
    p.check()
    _errors(False)


def test_fork_without_sharing():
    p = Pair()
    p.append([0, 1], [37, 32])
    p.c.fork([0, 1, 0], [2, 3, 4], share=False)
    p.m.fork([0, 1, 0], [2, 3, 4], share=False)
    p.check()
    p.c.free([0])
    p.m.free([0])
    p.append([2, 1], [40, 1])
    p.check()
    _errors(False)


def test_free_names_a_slot_twice():
    p = Pair()
    p.append([0, 1, 2], [20, 30, 40])
    p.c.fork([1], [4])
    p.m.fork([1], [4])
    p.c.free([1, 0, 1, 5, 1])
    p.m.free([1, 0, 1, 5, 1])
    p.check()
    _errors(False)


def test_compact():
    p = Pair(pages=60, slots=12)
    p.append([0, 1, 2, 3, 4, 5], [100, 20, 17, 64, 33, 1])
    p.c.fork([3], [6])
    p.m.fork([3], [6])
    p.c.free([0, 2])
    p.m.free([0, 2])
    p.c.compact()
    p.m.compact()
    p.check()
    assert p.c.free_pages() == sum(r == 0 for r in p.m.refs)
    p.c.compact()  # nothing to move
    p.check()
    p.append([0, 3, 6], [60, 3, 4])
    p.check()
    p.c.free(list(range(12)))
    p.m.free(list(range(12)))
    p.c.compact()  # nothing left
    p.m.compact()
    p.check()
    _errors(False)


@pytest.mark.parametrize("seed", range(4))
def test_random_steps(seed):
    """Appends, forks, frees and compactions in random order, pages often short."""
    import random
    r = random.Random(seed)
    p = Pair(pages=r.choice([30, 70]), page=16, slots=10, max_tokens=112, layers=1)
    failed = False
    for _ in range(60):
        kind = r.choice(["append"] * 4 + ["fork", "free", "compact"])
        m = p.m
        if kind == "append":
            slots = r.sample(range(10), r.randint(1, 6))
            new = [r.choice([0, 1, 1, 5, 16, 17, 40]) for _ in slots]
            p.append(slots, new)
            failed |= any(m.grown[s] != n for s, n in zip(slots, new))
        elif kind == "fork":
            empty = [s for s in range(10) if not m.lens[s]]
            full = [s for s in range(10) if m.lens[s]]
            if not empty or not full:
                continue
            dst = r.sample(empty, r.randint(1, len(empty)))
            src = [r.choice(full) for _ in dst]
            share = r.random() < 0.7
            before = [list(x) for x in m.rows]
            m.fork(src, dst, share)
            failed |= any(m.lens[b] != m.lens[a] for a, b in zip(src, dst)) and before is not None
            p.c.fork(src, dst, share)
        elif kind == "free":
            slots = [r.randrange(10) for _ in range(r.randint(1, 3))]
            p.c.free(slots)
            m.free(slots)
        else:
            p.c.compact()
            m.compact()
        from multi_gpu_flashattention_b200.ops.flash import KernelStatusError, check_errors
        try:
            check_errors()
        except KernelStatusError:
            assert failed
        p.check()


# ------------------------------------------------------------------ what goes wrong
def test_too_few_pages_leaves_the_sequence_as_it_was():
    p = Pair(pages=6, max_tokens=160)
    p.append([0, 1], [30, 16])
    p.append([2, 0, 1, 3], [1, 60, 16, 0])  # 1 + 2 + ... pages of the 3 left: 0 gets none
    p.check()
    assert p.m.grown[0] == 0 and p.m.lens[2] == 1
    _errors(True)
    p.c.fork([0, 1], [4, 5], share=False)
    p.m.fork([0, 1], [4, 5], share=False)
    p.check()
    _errors(True)


def test_row_too_short():
    p = Pair(max_tokens=40)  # three pages of 16
    p.append([0, 1], [48, 40])
    p.append([0, 1, 2], [1, 8, 5])
    p.check()
    assert p.m.grown[0] == 0 and p.m.lens[1] == 48
    _errors(True)


def test_slots_out_of_range_or_named_twice():
    p = Pair()
    p.append([0, 1], [20, 20])
    pos, _ = p.append([1, 12, -1, 1, 2], [3, 4, 5, 6, 7])
    assert pos[:3] == [20, 21, 22] and pos[-7:] == list(range(7))
    p.check()
    _errors(True)
    p.c.free([12, -3, 2])
    p.m.free([2])
    p.check()
    _errors(True)
    # a target that holds something, a target named twice, a source that is a target
    p.c.fork([0, 0, 1, 0, 3, 12], [1, 4, 4, 3, 5, 6])
    p.m.fork([0, 0], [4, 3])
    p.check()
    _errors(True)


def test_rows_of_refused_sequences():
    p = Pair(pages=6, layers=1)
    cu = [1, 4, 8, 28, 31, 31, 100, 103]
    slots = [3, 12, 1, 3, 0, 2, 5]   # slot 12 there is none, 3 again, 0 with no token, too many for 2
    p.c.reserve(slots, cu, 105)
    got = p.c.refused(slots, cu, 105)
    assert got.dtype == torch.bool
    want = torch.zeros(105, dtype=torch.bool)
    want[4:8] = want[28:31] = want[31:103] = True  # pages are given in order: 5 gets none
    assert p.c.lens.tolist()[:6] == [0, 20, 0, 3, 0, 0]
    assert torch.equal(got.cpu(), want)
    assert p.c.refused([], [0], 4).tolist() == [False] * 4 and p.c.refused([1], [0, 0], 0).shape == (0,)
    with pytest.raises(RuntimeError):
        p.c.refused([1], [0], 4)
    _errors(True)


@pytest.mark.parametrize("n", [1, 20])
def test_slot_named_twice_with_as_many_tokens(n):
    """The first naming's keys and values are the ones that are kept."""
    p = Pair(layers=1)
    p.append([0, 1], [5, 7])
    p.append([1, 0, 1, 2, 1], [n, 1, n, n, n])
    p.check()
    _errors(True)


def test_cu_seqlens_that_make_no_sense():
    p = Pair()
    p.append([0, 1], [20, 20])
    c = p.c
    c.reserve([0, 1, 2], [0, 5, 3, 9], 9)       # decreasing: sequence 1 is left out
    k = torch.zeros(9, H, D, device="cuda", dtype=torch.bfloat16)
    c.write(0, k, k, [0, 1, 2], [0, 5, 3, 9])
    assert c.lens.tolist()[:3] == [25, 20, 6]
    _errors(True)
    c.reserve([1], [0, 9], 4)                   # more than the batch has
    assert c.lens[1] == 20
    _errors(True)


def test_refusals():
    from multi_gpu_flashattention_b200 import PagedKVCache
    p = Pair()
    c = p.c
    k = torch.zeros(4, H, D, device="cuda", dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32, device="cuda")
    slots, cu = torch.tensor([0], **i32), torch.tensor([0, 4], **i32)
    for bad in (lambda: c.reserve(slots.long(), cu, 4), lambda: c.reserve(slots, cu[:1], 4),
                lambda: c.reserve(slots, cu, -1), lambda: c.reserve(slots.cpu(), cu, 4),
                lambda: c.write(2, k, k, slots, cu), lambda: c.write(-1, k, k, slots, cu),
                lambda: c.write(0, k.half(), k.half(), slots, cu), lambda: c.write(0, k, k[:3], slots, cu),
                lambda: c.write(0, k[:, :1], k[:, :1], slots, cu), lambda: c.write(0, k.cpu(), k.cpu(), slots, cu),
                lambda: c.fork(slots, cu), lambda: c.free(slots[None]),
                lambda: PagedKVCache.allocate(1, 4, 12, 1, 64, 2, 32),
                lambda: PagedKVCache.allocate(1, 4, 8, 1, 64, 2, 32),
                lambda: PagedKVCache.allocate(1, 4, 16, 1, 96, 2, 32),
                lambda: PagedKVCache.allocate(1, 4, 16, 1, 64, 2, 32, dtype=torch.float32),
                lambda: PagedKVCache(c.k, c.v[:1], c.page_table, c.lens, c.refs, c.grown),
                lambda: PagedKVCache(c.k, c.v, c.page_table.t(), c.lens, c.refs, c.grown),
                lambda: PagedKVCache(c.k, c.v, c.page_table, c.lens, c.refs[1:], c.grown)):
        with pytest.raises(RuntimeError):
            bad()
    c.reserve([], [0], 0)
    c.free([])
    c.fork([], [])
    p.check()
    _errors(False)


def test_counts_beyond_32_bits_are_refused():
    """Where the sums of pages, tiles and tokens would not fit (memory is reserved, not touched)."""
    from multi_gpu_flashattention_b200 import PagedKVCache, paged_attention
    c = Pair().c
    i32 = dict(dtype=torch.int32, device="cuda")
    zeros = lambda n: torch.zeros(n, **i32)
    with pytest.raises(RuntimeError, match="out of range"):
        c.reserve([0], [0, 1], 1 << 30)
    with pytest.raises(RuntimeError, match="too many entries"):
        PagedKVCache(c.k, c.v, torch.empty(4096, 1 << 19, **i32), zeros(4096), c.refs, zeros(4096))
    # 257 sequences of 2^24 tiles of 64 keys: nothing is computed, and the error is reported
    k = torch.zeros(2, 1024, H, D, device="cuda", dtype=torch.bfloat16)
    wide = zeros((1 << 20) - 1)[None]
    q = torch.zeros(257, H, D, device="cuda", dtype=torch.bfloat16)
    out = torch.ones_like(q)
    for lens, wrong in ((0, False), (wide.numel() * 1024, True)):
        paged_attention(q, k, k, wide, zeros(1) + lens, torch.arange(258, **i32), 1, slots=zeros(257), out=out)
        _errors(wrong)
        assert (out == 0).all()                 # of the empty sequences


def test_an_error_is_raised_by_the_next_call(monkeypatch):
    monkeypatch.undo()
    from multi_gpu_flashattention_b200.ops.flash import KernelStatusError
    p = Pair(pages=2)
    p.c.reserve([0], [0, 33], 33)
    torch.cuda.synchronize()
    with pytest.raises(KernelStatusError, match="too few free pages"):
        p.c.free([0])
    p.c.free([0])


# ------------------------------------------------------------------ as it is used
def test_strided_pools_and_inputs():
    """Keys and values of one pool, heads before tokens; new ones cut from a projection."""
    from multi_gpu_flashattention_b200 import PagedKVCache
    p = Pair()
    pool = torch.full((2, 40, 2, H, 16, D), float("nan"), device="cuda", dtype=torch.bfloat16)
    k, v = (pool[:, :, i].transpose(2, 3) for i in (0, 1))
    p.c = PagedKVCache(k, v, p.c.page_table, p.c.lens, p.c.refs, p.c.grown)
    p.append([0, 1], [37, 20])
    p.c.fork([0], [3])
    p.m.fork([0], [3])
    p.c.free([0])
    p.m.free([0])
    p.c.compact()
    p.m.compact()
    p.check()
    wide = torch.cat([_value([900, 901, 902], 0, 0), _value([900, 901, 902], 0, 1)], 1)
    p.c.reserve([5], [0, 3], 3)
    p.m.reserve([5], [3])
    p.c.write(0, wide[:, :H], wide[:, H:], [5], [0, 3])
    row = p.m.rows[5][0]
    assert torch.equal(p.c.k[0, row, :3], wide[:, :H]) and torch.equal(p.c.v[0, row, :3], wide[:, H:])


def test_steps_in_a_graph_and_on_a_stream():
    """A decode step (reserve, write, attend) captured once and replayed token by token,
    against the same steps made eagerly."""
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    i32 = dict(dtype=torch.int32, device="cuda")
    slots, cu = torch.tensor([2, 0, 5], **i32), torch.tensor([0, 1, 2, 3], **i32)
    g = torch.Generator("cuda").manual_seed(0)
    steps = [torch.randn(3, 8, D, device="cuda", generator=g).bfloat16() for _ in range(20)]
    outs = []
    for graphed in (False, True):
        p = Pair(layers=1)
        p.append([2, 0, 5], [15, 3, 31])
        x = steps[0].clone()

        def step():
            pos = p.c.reserve(slots, cu, 3)
            p.c.write(0, x[:, :H], x[:, H:2 * H], slots, cu)
            return pos, p.c.attend(0, x[:, 4:], slots, cu, 1)

        got = []
        if graphed:
            saved = [t.clone() for t in (p.c.page_table, p.c.lens, p.c.refs, p.c.grown)]
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step()
                for t, u in zip((p.c.page_table, p.c.lens, p.c.refs, p.c.grown), saved):
                    t.copy_(u)
            torch.cuda.current_stream().wait_stream(s)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
        for data in steps:
            x.copy_(data)
            if graphed:
                graph.replay()
            else:
                out = step()
            got.append([t.clone() for t in out])
        check_errors()
        outs.append(got)
        assert p.c.lens.tolist()[:6] == [23, 0, 35, 0, 0, 51]
    for a, b in zip(*outs):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
