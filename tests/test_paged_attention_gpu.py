"""paged_attention against plain attention in 64 bits.

Tolerances, fixed before the first run. The output is a mean of values with weights p
that sum to one: it is rounded once to its type (u of the value, u = finfo.eps / 2), and
the weights are rounded to 16 bits (u each: u * sum p |v|, which bounds any order of
signs); scores, sums and maxima are fp32 (scores of 128 products of 16-bit numbers, and
2^x to 2^-22: below 2e-5 relative on a weight for scores up to 40). So |error| <=
u |out| + (u + 4e-5) sum p |v| + 2^-25 (fp16's smallest steps). The LSE has no 16-bit
rounding: 2e-5 (1 + |lse|).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


class Problem:
    """Sequences with `new` new tokens at the end of `kv`, in pages in random order; what
    is behind a sequence's end, and every page of nobody, is NaN."""

    def __init__(self, new, kv, heads, kv_heads, D, page, dtype=torch.bfloat16, seed=0, spare=3,
                 tail=0, big=1.0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.new, self.kv, self.page, self.dtype = new, kv, page, dtype
        need = [-(-n // page) for n in kv]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        width = max(max(need), 1)
        table, at = [], 0
        self.k = torch.full((pages, page, kv_heads, D), float("nan"), device="cuda", dtype=dtype)
        self.v = torch.full_like(self.k, float("nan"))
        self.keys, self.values = [], []
        for n, m in zip(kv, need):
            ids = order[at:at + m]
            at += m
            table.append(ids + [-1] * (width - m))
            a = (torch.randn(n, kv_heads, D, device="cuda", generator=g) * big).to(dtype)
            b = torch.randn(n, kv_heads, D, device="cuda", generator=g).to(dtype)
            self.keys.append(a)
            self.values.append(b)
            for j, i in enumerate(ids):
                part = slice(j * page, min(n, (j + 1) * page))
                self.k[i, :part.stop - part.start] = a[part]
                self.v[i, :part.stop - part.start] = b[part]
        i32 = dict(dtype=torch.int32, device="cuda")
        self.table = torch.tensor(table, **i32).view(len(kv), width)
        self.lens = torch.tensor(kv, **i32)
        self.cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], **i32)
        self.q = (torch.randn(sum(new) + tail, heads, D, device="cuda", generator=g) * big).to(dtype)
        self.max_new = max(new) if new else 0

    def run(self, **kw):
        from multi_gpu_flashattention_b200 import paged_attention
        kw.setdefault("return_lse", True)
        return paged_attention(self.q, self.k, self.v, self.table, self.lens, self.cu,
                               kw.pop("max_new", self.max_new), **kw)

    def check(self, out, lse, causal=True, scale=None):
        u = torch.finfo(self.dtype).eps / 2
        heads, D = self.q.shape[1:]
        for b, (n, kv) in enumerate(zip(self.new, self.kv)):
            if n == 0:
                continue
            rows = slice(int(self.cu[b]), int(self.cu[b + 1]))
            k, v = (t.double().repeat_interleave(heads // t.shape[1], 1) for t in (self.keys[b], self.values[b]))
            s = torch.einsum("qhd,khd->hqk", self.q[rows].double(), k) * (scale or 1 / math.sqrt(D))
            if causal:
                last = torch.arange(n, device="cuda") + kv - n
                s.masked_fill_(torch.arange(kv, device="cuda") > last[:, None], float("-inf"))
            ref_lse = torch.logsumexp(s, -1)
            p = torch.nan_to_num(torch.exp(s - ref_lse[..., None]))
            ref = torch.einsum("hqk,khd->qhd", p, v)
            size = torch.einsum("hqk,khd->qhd", p, v.abs())
            err = (out[rows].double() - ref).abs()
            bound = u * ref.abs() + (u + 4e-5) * size + 2.0 ** -25
            assert (err <= bound).all(), f"sequence {b}: out off by {err.max().item()} " \
                f"({int((~(err <= bound)).sum())} of {err.numel()})"
            got = lse[:, rows].double()
            dead = ref_lse == float("-inf")
            assert (got[dead] == float("-inf")).all() and not out[rows].transpose(0, 1)[dead].any()
            e = (got - ref_lse)[~dead].abs()
            assert (e <= 2e-5 * (1 + ref_lse[~dead].abs())).all(), f"sequence {b}: lse off by {e.max().item()}"


def _both(p, **kw):
    for causal in (True, False):
        out, lse = p.run(causal=causal, **kw)
        p.check(out, lse, causal)


# ------------------------------------------------------------------ single tokens
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,D,page", [(4, 4, 64, 16), (8, 2, 128, 16), (7, 1, 128, 64),
                                                   (32, 8, 128, 32), (16, 1, 64, 128), (32, 1, 128, 256)])
def test_one_token(heads, kv_heads, D, page, dtype):
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000]
    _both(Problem([1] * len(kv), kv, heads, kv_heads, D, page, dtype))


@pytest.mark.parametrize("kv", [[5000], [20011, 3], [1, 1, 1, 9000], [4096] * 3])
def test_one_token_split_over_ctas(kv):
    _both(Problem([1] * len(kv), kv, 8, 2, 128, 64))


def test_one_token_full_batch():
    g = torch.Generator().manual_seed(5)
    kv = torch.randint(1, 2000, (300,), generator=g).tolist()
    _both(Problem([1] * 300, kv, 8, 2, 64, 16))


@pytest.mark.parametrize("new", [2, 3, 4, 8])
def test_few_tokens(new):
    """Up to 32 rows a key head: some tokens see fewer keys than others."""
    kv = [new, new + 1, 16, 70, 500, 2048]
    kv = [max(new, n) for n in kv]
    _both(Problem([new] * len(kv), kv, 8, 2, 128, 16))
    mixed = [new, 1, 0, new - 1, new, 1]
    _both(Problem(mixed, kv, 4, 1, 64, 32))


# ------------------------------------------------------------------ chunks
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,D,page", [(4, 4, 64, 16), (8, 2, 128, 16), (7, 1, 128, 64),
                                                   (6, 2, 64, 128), (32, 8, 128, 256), (16, 1, 128, 32)])
def test_chunk(heads, kv_heads, D, page, dtype):
    new = [1, 40, 128, 129, 200, 333]
    kv = [1, 40, 300, 129, 1500, 340]
    _both(Problem(new, kv, heads, kv_heads, D, page, dtype))


@pytest.mark.parametrize("group", [1, 5, 33, 64, 65, 100, 128])
def test_chunk_group_sizes(group):
    """Groups that fill a tile, do not divide it, or leave a token a tile."""
    _both(Problem([35, 3], [100, 200], group, 1, 64, 16))


@pytest.mark.parametrize("n", [9, 10, 17, 31])
def test_chunk_of_fewer_tokens_than_a_tile(n):
    _both(Problem([n], [n + 700], 4, 1, 128, 64))
    _both(Problem([n], [n + 3000], 8, 2, 64, 16))


def test_chunk_split_over_ctas():
    _both(Problem([64], [30000], 4, 1, 128, 64))
    _both(Problem([200, 50], [9000, 60], 8, 2, 128, 16))


def test_chunk_long():
    _both(Problem([1500, 700, 2], [1500, 4000, 2], 4, 2, 128, 64))


def test_many_units_per_cta():
    _both(Problem([90] * 40, [95 + i for i in range(40)], 8, 8, 64, 16))


@pytest.mark.parametrize("new,kv", [([128] * 40, [128] * 40), ([64] * 200, [64] * 199 + [1100]),
                                    ([256] * 2, [8000] * 2), ([24] * 3, [5000, 300, 24]),
                                    ([1, 40, 128, 129, 200, 333], [1, 40, 300, 129, 1500, 340])])
def test_again_between_other_kernels(new, kv):
    """The same call on SMs whose registers and memories other kernels have used since."""
    p = Problem(new, kv, 32, 8, 128, 64)
    want, want_lse = p.run()
    p.check(want, want_lse)
    for _ in range(4):
        x = torch.randn(1500, 1500, device="cuda", dtype=torch.float64)
        int(((x @ x).abs().amax(-1) > 1e9).sum())
        out, lse = p.run()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_chunk_kernel_spills_nothing():
    """Its launch refuses a build in which a score could be spilled while it is being loaded."""
    from multi_gpu_flashattention_b200._ext import C
    assert C().paged_chunk_local_bytes() == 0


@pytest.mark.parametrize("new,kv", [([100] * 64, [100] * 64), ([40, 0, 33, 1], [300, 5, 33, 900])])
def test_max_seqlen_far_above_the_longest(new, kv):
    """Short tables, whose units are dealt out by max_seqlen_q where it is close."""
    p = Problem(new, kv, 4, 2, 64, 16)
    for most in (max(new), 8 * max(new), sum(new), 1 << 40):
        out, lse = p.run(max_new=most)
        p.check(out, lse)


def test_max_seqlen_that_only_bounds_the_batch_costs_little():
    """512 chunks of 100 tokens over 100 keys, announced as up to 51200 tokens each."""
    p = Problem([100] * 512, [100] * 512, 32, 8, 128, 64)
    times = {}
    for most in (100, sum(p.new)):
        p.run(max_new=most)
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        best = float("inf")
        for _ in range(5):
            a.record()
            p.run(max_new=most)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        times[most] = best
    assert times[51200] < 3 * times[100], times  # it was 23 times as long


# ------------------------------------------------------------------ rows and masks
@pytest.mark.parametrize("new,heads", [([4, 3], 4), ([60, 50], 4)])
def test_tokens_without_a_visible_key(new, heads):
    """More new tokens than keys (the first see none), and sequences without keys."""
    p = Problem(new + [1, 2], [2, 0, 0, 1], heads, 1, 128, 16)
    out, lse = p.run()
    p.check(out, lse)
    out, lse = p.run(causal=False)
    p.check(out, lse, causal=False)


@pytest.mark.parametrize("max_new", [1, 64])
def test_rows_outside_every_sequence_are_left(max_new):
    new = [1, 0, 1] if max_new == 1 else [64, 0, 3]
    p = Problem(new, [100, 7, 200], 4, 2, 64, 16, tail=9)
    out = torch.full_like(p.q, 77.0)
    got, lse = p.run(out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (out[sum(new):] == 77.0).all()
    p.check(out, lse)


@pytest.mark.parametrize("new", [1, 50])
def test_large_scores(new):
    """Scores far apart: the maximum moves along the run."""
    p = Problem([new], [3000], 4, 2, 64, 16, big=2.0)
    out, lse = p.run(softmax_scale=0.35)
    p.check(out, lse, scale=0.35)


class Shared(Problem):
    """`seqs` sequences over the same pages, with keys (x, 0, ..., 0) for x of `first`, and
    queries (1, 0, ..., 0), so that scores are x * scale; enough of them that a CTA goes
    over a sequence's keys without a cut."""

    def __init__(self, first, values, new, seqs, dtype):
        super().__init__([new], [first.numel()], 1, 1, 64, 64, dtype)
        self.new, self.kv = [new] * seqs, [first.numel()] * seqs
        k = torch.zeros(first.numel(), 1, 64, device="cuda", dtype=dtype)
        k[:, 0, 0] = first
        v = values[:, None, None].expand(-1, 1, 64).to(dtype)
        for t, pool in ((k, self.k), (v, self.v)):
            for j, i in enumerate(self.table[0].tolist()):
                part = t[j * 64:(j + 1) * 64]
                pool[i, :part.shape[0]] = part
        self.keys, self.values = [k] * seqs, [v] * seqs
        self.table = self.table.expand(seqs, -1).contiguous()
        self.lens = self.lens.expand(seqs).contiguous()
        self.cu = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * new
        self.q = torch.zeros(seqs * new, 1, 64, device="cuda", dtype=dtype)
        self.q[..., 0] = 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at", [0, 20000])
@pytest.mark.parametrize("new,seqs", [(1, 320), (40, 160)])
def test_many_small_weights_beside_a_large_one(new, seqs, at, dtype):
    """One key with the value 0 and 32767 with the value 1 and 2^-25.2 of its weight, which
    fp16 has no step for. Beyond the tolerance of a weight's relative rounding, an fp16 weight
    may be off by 2^-36 of the largest: fp16's step at its small end, 2^-24, is 2^-35 of the
    2^11 that the largest is given at least."""
    n = 32768
    first, values = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    first[at], values[at] = 16.0, 0.0
    p = Shared(first, values, new, seqs, dtype)
    out, lse = p.run(causal=False, softmax_scale=25.2 * math.log(2) / 16)
    w = 2.0 ** -25.2
    total = 1 + (n - 1) * w
    want, u = (n - 1) * w / total, torch.finfo(dtype).eps / 2
    bound = u * want + (u + 4e-5) * want + (n - 1) * 2.0 ** -36 + 2.0 ** -25
    assert (out.double() - want).abs().max().item() <= bound
    ref = 25.2 * math.log(2) + math.log(total)
    assert (lse.double() - ref).abs().max().item() <= 2e-5 * (1 + ref)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step", [0.4, 1.7, 3.9, 4.1, 8.1])
@pytest.mark.parametrize("new,seqs", [(1, 320), (40, 160)])
def test_a_maximum_that_creeps_up(new, seqs, step, dtype):
    """Scores that grow by `step` powers of two every 128 keys: by less and by more than a
    kernel lets its maximum lag. No weight may pass the type's largest number."""
    n = 8000
    tile = torch.arange(n, device="cuda") // 128
    g = torch.Generator("cuda").manual_seed(3)
    p = Shared(tile.float(), torch.randn(n, device="cuda", generator=g), new, seqs, dtype)
    scale = step * math.log(2)
    out, lse = p.run(causal=False, softmax_scale=scale)
    p.check(out, lse, causal=False, scale=scale)


@pytest.mark.parametrize("new", [1, 40])
def test_nan_in_a_query_stays_in_its_row(new):
    p = Problem([new, new], [90, 300], 4, 2, 64, 16)
    clean, clean_lse = p.run()
    p.q[new - 1, 1, 3] = float("nan")
    out, lse = p.run()
    assert out[new - 1, 1].isnan().all() and lse[1, new - 1].isnan()
    out[new - 1, 1], lse[1, new - 1] = clean[new - 1, 1], clean_lse[1, new - 1]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


# ------------------------------------------------------------------ layouts
@pytest.mark.parametrize("new", [1, 70])
def test_strides(new):
    """q cut from a wider projection, pages with heads first, keys and values of one
    pool, an output with strides, a table with more rows than sequences."""
    p = Problem([new, new], [new + 100, new + 5], 8, 2, 128, 32)
    want, want_lse = p.run()
    p.check(want, want_lse)
    wide = torch.zeros(p.q.shape[0], 12, 128, device="cuda", dtype=p.dtype)
    wide[:, 2:10] = p.q
    p.q = wide[:, 2:10]
    pool = torch.stack([p.k, p.v], 1)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (p.k, p.v)]
    room = torch.zeros_like(wide)
    for k, v in ((pool[:, 0], pool[:, 1]), heads_first):
        p.k, p.v = k, v
        out, lse = p.run(out=room[:, :8])
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    rows = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    table = torch.full((5, p.table.shape[1]), -1, dtype=torch.int32, device="cuda")
    lens = torch.full((5,), 1 << 20, dtype=torch.int32, device="cuda")
    table[rows.long()], lens[rows.long()] = p.table, p.lens
    p.table, p.lens = table, lens
    out, lse = p.run(slots=rows)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("new", [1, 48])
def test_same_result_every_time_and_on_two_streams(new):
    p = Problem([new] * 5, [700, 50, 5000, 51, 1200], 8, 2, 128, 16)
    want, lse = p.run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(p.run())
    torch.cuda.synchronize()
    for o, l in got:
        assert torch.equal(o, want) and torch.equal(l, lse)


@pytest.mark.parametrize("new", [1, 48])
def test_graph_with_lengths_that_change(new):
    """A captured call follows the lengths and the table; two graphs run side by side."""
    p = Problem([new] * 3, [900, 800, 700], 8, 2, 64, 16)
    p.run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(p.run())
        graphs.append(g)
    other = Problem([new] * 3, [new, 333, 40 + new], 8, 2, 64, 16, seed=9)
    other.k, other.v, other.q = p.k, p.v, p.q
    for b, n in enumerate(other.kv):
        p.lens[b] = n
        other.keys[b], other.values[b] = p.keys[b][:n], p.values[b][:n]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for out, lse in outs:
        other.check(out, lse)


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes, used at its far end."""
    pages, page, D = 300, 1024, 128
    k = torch.empty(pages, page, 64, D, dtype=torch.bfloat16, device="cuda")  # 5 GB
    p = Problem([1, 40], [900, 950], 2, 1, D, 1024, spare=0)
    at = [pages - 1, pages - 2]
    for i in range(2):
        k[at[i], :, 60] = p.k[p.table[i, 0]][:, 0]
        k[at[i], :, 61] = p.v[p.table[i, 0]][:, 0]
    p.k, p.v = k[:, :, 60:61], k[:, :, 61:62]
    p.table = torch.tensor([[at[0]], [at[1]]], dtype=torch.int32, device="cuda")
    out, lse = p.run()
    p.check(out, lse)


# ------------------------------------------------------------------ refusals and errors
def test_refusals():
    from multi_gpu_flashattention_b200 import paged_attention
    p = Problem([1, 1], [20, 30], 8, 2, 64, 16)
    base = dict(q=p.q, k=p.k, v=p.v, table=p.table, lens=p.lens, cu=p.cu, max_new=1)

    def call(kw=None, **over):
        a = dict(base, **over)
        return paged_attention(a["q"], a["k"], a["v"], a["table"], a["lens"], a["cu"], a["max_new"], **(kw or {}))

    call()
    odd = torch.zeros(2, 8, 65, device="cuda", dtype=p.dtype)[..., 1:]
    for over in (dict(q=p.q.float()), dict(q=p.q.half()), dict(q=p.q[:, :7]), dict(q=p.q.cpu()), dict(q=odd),
                 dict(q=p.q[..., :32]), dict(k=p.k[:, :12], v=p.v[:, :12]), dict(k=p.k[:, :8], v=p.v[:, :8]),
                 dict(v=p.v[:2]), dict(table=p.table.long()), dict(table=p.table[:1]), dict(lens=p.lens[:1]),
                 dict(lens=p.lens.cpu()), dict(cu=p.cu.long()), dict(cu=p.cu[None]), dict(max_new=-1),
                 dict(q=p.q[:1].expand(2, 8, 64)),
                 dict(kw=dict(softmax_scale=0.0)), dict(kw=dict(softmax_scale=-1.0)),
                 dict(kw=dict(out=p.q[:1])), dict(kw=dict(out=p.q.half())), dict(kw=dict(slots=p.cu)),
                 dict(kw=dict(status=torch.zeros(1, dtype=torch.int32)))):
        with pytest.raises(RuntimeError):
            call(**over)
    with pytest.raises(RuntimeError, match="no gradient"):
        call(q=p.q.clone().requires_grad_())
    with torch.no_grad():
        call(q=p.q.clone().requires_grad_())


def test_scales_outside_float32_are_refused():
    """As a float they are 0 or infinite, and 0 times a hidden score is NaN."""
    p = Problem([1], [30], 4, 2, 64, 16)
    for scale in (1e-50, 1e39, float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="softmax_scale must be positive"):
            p.run(softmax_scale=scale)
    out, lse = p.run(softmax_scale=1e-30)
    p.check(out, lse, scale=1e-30)


@pytest.mark.parametrize("pinned", [False, True])
def test_a_status_word_of_the_caller(pinned):
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    p = Problem([1], [30], 4, 2, 64, 16)
    word = torch.zeros(1, dtype=torch.int32)
    word = word.pin_memory() if pinned else word.cuda()
    out, lse = p.run(status=word)
    p.check(out, lse)
    assert int(word) == 0
    p.table[0, 0] = -1
    p.run(status=word)
    torch.cuda.synchronize()
    assert int(word) & 0xff == 4
    check_errors()


@pytest.mark.multigpu
def test_a_status_word_of_another_device_is_refused():
    p = Problem([1], [30], 4, 2, 64, 16)
    with pytest.raises(RuntimeError, match="status must be on q's device"):
        p.run(status=torch.zeros(1, dtype=torch.int32, device="cuda:1"))


@pytest.mark.parametrize("new", [1, 40])
def test_wrong_contents_are_reported(new):
    """Pages that are not in the pool, lengths beyond the table, slots out of range, rows
    out of range: an error word, no fault, and the other sequences are right."""
    from multi_gpu_flashattention_b200.ops.flash import KernelStatusError, check_errors

    def wrong(change):
        p = Problem([new, new], [new + 60, new + 90], 4, 2, 64, 16)
        slots = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        kw = change(p, slots) or {}
        out, lse = p.run(slots=slots, **kw)
        with pytest.raises(KernelStatusError):
            check_errors()
        check_errors()  # re-armed
        p.new, p.cu = [0, new], torch.tensor([0, new, 2 * new])
        p.check(out, lse)

    def entry(v):
        return lambda p, s: p.table[0].__setitem__(1, v)

    wrong(entry(-1))
    wrong(entry(1 << 30))
    wrong(lambda p, s: p.lens.__setitem__(0, 1 << 30))
    wrong(lambda p, s: p.lens.__setitem__(0, -5))
    wrong(lambda p, s: s.__setitem__(0, 2))
    wrong(lambda p, s: s.__setitem__(0, -1))


def test_more_tokens_than_announced_are_reported():
    from multi_gpu_flashattention_b200.ops.flash import KernelStatusError, check_errors
    p = Problem([3, 1], [60, 90], 4, 2, 64, 16)
    out = torch.full_like(p.q, 5.0)
    p.run(out=out, max_new=1)
    with pytest.raises(KernelStatusError):
        check_errors()
    assert (out[:3] == 5.0).all()
    p = Problem([40, 40], [60, 90], 4, 2, 64, 16)
    p.cu[2] = 10000
    p.run()
    with pytest.raises(KernelStatusError):
        check_errors()


def test_rows_beyond_32_bits():
    """Tokens times query heads a key head pass 2^31 (overlapping rows, none of them used)."""
    tokens, heads = 1 << 25, 64
    q = torch.zeros(tokens * 8 + heads * 64, device="cuda", dtype=torch.bfloat16)
    q = q.as_strided((tokens, heads, 64), (8, 64, 1))
    p = Problem([1], [30], 64, 1, 64, 16)
    p.q, p.max_new = q, tokens
    p.cu.zero_()
    p.run(out=q, return_lse=False)
    assert not q[::1 << 20].any()


def test_empty_batches():
    p = Problem([0, 0], [5, 6], 4, 2, 64, 16, tail=3)
    out = torch.full_like(p.q, 3.0)
    p.run(out=out, max_new=1)
    assert (out == 3.0).all()
    p.cu = p.cu[:1]
    p.run(max_new=1)
    p = Problem([1], [5], 4, 2, 64, 16)
    p.q = p.q[:0]
    p.cu.zero_()
    out, lse = p.run()
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
