"""The decoder's operators together, as a model uses them: served over a paged cache and
trained with the fused norms and rotary positions, against the same model in 64 bits.

The bound: the kernels round no more often than the model's plain 16-bit operators do (a
norm rounds once and not twice, a rotation once, attention as flash_attn does), so the
distance from the 64-bit model is at most that of the plain 16-bit model, up to the
chance of the individual roundings, for which half as much again is allowed.
"""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

VOCAB, DIM, LAYERS, HEADS, KV, D = 97, 256, 3, 4, 2, 64


def _model(dtype, fused=False, seed=0):
    from multi_gpu_flashattention_b200 import RingTransformerLM
    torch.manual_seed(seed)
    m = RingTransformerLM(VOCAB, DIM, LAYERS, HEADS, KV, head_dim=D, mlp_mult=2, fused_ops=fused)
    torch.nn.init.normal_(m.embed.weight, std=0.5)
    for blk in m.blocks:
        for n in (blk.norm1, blk.norm2):
            torch.nn.init.normal_(n.weight, 1.0, 0.2)
    return m.to("cuda", dtype)


def _exact(model, ids):
    """Logits of ids [S] from the parameters in 64 bits, with differentiable copies."""
    P = {n: p.detach().double().requires_grad_() for n, p in model.named_parameters()}
    P.setdefault("head.weight", P["embed.weight"])
    norm = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    S = ids.numel()
    ang = torch.arange(S, device="cuda", dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]

    def rot(t):
        a, b = t.split(D // 2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    x = P["embed.weight"][ids]
    hide = torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1)
    for i in range(LAYERS):
        W = lambda n: P[f"blocks.{i}.{n}.weight"]
        h = norm(x, W("norm1"))
        q, k, v = ((h @ W(n).t()).view(S, -1, D) for n in ("wq", "wk", "wv"))
        q, k = rot(q), rot(k)
        k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) / D ** 0.5
        a = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(hide, float("-inf")), -1), v)
        x = x + a.reshape(S, -1) @ W("wo").t()
        h = norm(x, W("norm2"))
        x = x + (F.silu(h @ W("w1").t()) * (h @ W("w3").t())) @ W("w2").t()
    return norm(x, P["norm.weight"]) @ P["head.weight"].t(), P


def _ids(n, seed):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


def _plain(model, ids):
    from multi_gpu_flashattention_b200 import RingLayout
    lay = RingLayout("contiguous", ids.numel(), 1, mask="causal")
    return model(ids[None], lay)[0]


def _off(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


def _batch(parts):
    i32 = dict(dtype=torch.int32, device="cuda")
    cu = [0]
    for p in parts:
        cu.append(cu[-1] + p.numel())
    return torch.cat(parts), torch.tensor(cu, **i32), max(p.numel() for p in parts)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_serving_matches_the_model(dtype):
    """Three prompts in ragged chunks, then token by token, one of them forked on the way,
    the pool compacted once: all logits against the whole sequences at once."""
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    model = _model(dtype)
    seqs = [_ids(150, 1), _ids(70, 2), _ids(33, 3)]
    tail = _ids(12, 4)
    seqs.append(torch.cat([seqs[0][:100], tail]))      # forked from sequence 0 after 100 tokens
    want = [_exact(model, s)[0].detach() for s in seqs]
    with torch.no_grad():
        plain = max(_off(_plain(model, s), w) for s, w in zip(seqs, want))
    cache = model.make_cache(pages=40, page_size=16, slots=6, max_tokens=160)
    slot, done, got = [4, 0, 2, 5], [0, 0, 0, 100], [[], [], [], []]

    def step(which, n):
        parts = [seqs[b][done[b]:done[b] + k] for b, k in zip(which, n)]
        ids, cu, most = _batch(parts)
        slots = torch.tensor([slot[b] for b in which], dtype=torch.int32, device="cuda")
        out = model.serve(ids, cache, slots, cu, most)
        for i, (b, k) in enumerate(zip(which, n)):
            got[b].append(out[int(cu[i]):int(cu[i + 1])])
            done[b] += k

    step([0, 1, 2], [64, 5, 1])
    step([2, 0, 1], [30, 36, 40])
    cache.fork([slot[0]], [slot[3]])
    step([3, 0, 1, 2], [1, 1, 20, 2])
    step([0, 3], [17, 9])
    cache.compact()
    while any(done[b] < seqs[b].numel() for b in range(4)):
        live = [b for b in range(4) if done[b] < seqs[b].numel()]
        step(live, [1] * len(live))
    check_errors()
    got[3].insert(0, torch.cat(got[0])[:100])
    for b in range(4):
        off = _off(torch.cat(got[b]), want[b])
        assert off <= 1.5 * plain, f"sequence {b}: {off} of the norm, the plain model {plain}"
    cache.free([slot[b] for b in range(4)])
    assert cache.free_pages() == 40
    check_errors()


def test_training_with_fused_operators():
    """Loss and gradients of the fused model, as far from 64 bits as the plain one."""
    ids = _ids(257, 7)
    offs = {}
    for fused in (False, True):
        model = _model(torch.bfloat16, fused)
        loss = F.cross_entropy(_plain(model, ids[:-1]).float(), ids[1:])
        loss.backward()
        logits, P = _exact(model, ids[:-1])
        ref = F.cross_entropy(logits, ids[1:])
        names = [n for n, _ in model.named_parameters()]
        grads = torch.autograd.grad(ref, [P[n] for n in names])
        offs[fused] = {n: _off(p.grad, g) for (n, p), g in zip(model.named_parameters(), grads)}
        offs[fused]["loss"] = abs(loss.item() - ref.item()) / ref.item()
    plain = sum(offs[False].values()) / len(offs[False])
    for n, o in offs[True].items():
        assert o <= 1.5 * max(offs[False][n], plain), (n, o, offs[False][n], plain)


def test_fused_operators_leave_the_plain_model_alone():
    model = _model(torch.bfloat16)
    ids = _ids(64, 9)
    assert not model.fused_ops
    a = _plain(model, ids)
    model.fused_ops = True
    for b in model.blocks:
        b.fused_ops = True
    assert a.shape == _plain(model, ids).shape


def test_serving_steps_without_tokens():
    """No sequence at all, and sequences that get no token: empty logits, an unchanged cache."""
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    model = _model(torch.bfloat16)
    cache = model.make_cache(pages=8, page_size=16, slots=3, max_tokens=64)
    i32 = dict(dtype=torch.int32, device="cuda")
    prompt = _ids(20, 5)
    model.serve(prompt, cache, torch.tensor([1], **i32), torch.tensor([0, 20], **i32), 20)
    for slots, cu in (([], [0]), ([1, 2], [0, 0, 0])):
        out = model.serve(prompt[:0], cache, torch.tensor(slots, **i32), torch.tensor(cu, **i32), 0)
        assert out.shape == (0, VOCAB) and cache.lens.tolist() == [0, 20, 0]
    check_errors()


def test_training_with_fused_operators_under_autocast():
    """A stream in 32 bits, products in 16: gradients as far from 64 bits as the plain model's."""
    ids = _ids(130, 11)
    offs = {}
    for fused in (False, True):
        model = _model(torch.float32, fused)
        with torch.autocast("cuda", torch.bfloat16):
            out = _plain(model, ids[:-1])
        F.cross_entropy(out.float(), ids[1:]).backward()
        logits, P = _exact(model, ids[:-1])
        names = [n for n, _ in model.named_parameters()]
        grads = torch.autograd.grad(F.cross_entropy(logits, ids[1:]), [P[n] for n in names])
        offs[fused] = {n: _off(p.grad, g) for (n, p), g in zip(model.named_parameters(), grads)}
    plain = sum(offs[False].values()) / len(offs[False])
    for n, o in offs[True].items():
        assert o <= 1.5 * max(offs[False][n], plain), (n, o, offs[False][n], plain)


def test_a_sequence_without_room_leaves_the_others_whole(monkeypatch):
    """One of a step's sequences gets no pages, and its error is known before the first
    layer's write: the others' logits, keys and values are those of a step in which all had
    room, and the refused sequence is served once there is."""
    from multi_gpu_flashattention_b200 import KernelStatusError, PagedKVCache
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    model = _model(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device="cuda")
    slots = torch.tensor([0, 1, 2], **i32)
    first, cu1, most1 = _batch([_ids(20, 1), _ids(3, 2), _ids(10, 3)])
    ids, cu, most = _batch([_ids(1, 4), _ids(40, 5), _ids(6, 6)])  # 0, 2 and 0 pages more
    write = PagedKVCache.write

    def late(self, *a):  # what reserve() reported has arrived
        torch.cuda.synchronize()
        return write(self, *a)

    monkeypatch.setattr(PagedKVCache, "write", late)
    runs = {}
    for pages in (16, 5):
        cache = model.make_cache(pages=pages, page_size=16, slots=4, max_tokens=96)
        model.serve(first, cache, slots, cu1, most1)
        torch.cuda.synchronize()
        check_errors()
        runs[pages] = model.serve(ids, cache, slots, cu, most), cache
    (got, short), (want, roomy) = runs[5], runs[16]
    with pytest.raises(KernelStatusError, match="too few free pages"):
        model.serve(ids[1:41], short, slots[1:2], torch.tensor([0, 40], **i32), 40)
    assert short.lens.tolist() == [21, 3, 16, 0] and roomy.lens.tolist() == [21, 43, 16, 0]
    check_errors()
    for rows in (slice(0, 1), slice(41, 47)):
        assert torch.equal(got[rows], want[rows])

    def held(cache, slot):
        n = int(cache.lens[slot])
        rows = cache.page_table[slot, :-(-n // 16)].long()
        return [pool[:, rows].flatten(1, 2)[:, :n] for pool in (cache.k, cache.v)]

    for slot in (0, 2):
        for a, b in zip(held(short, slot), held(roomy, slot)):
            assert torch.equal(a, b)
    short.free([0])
    again = model.serve(ids[1:41], short, slots[1:2], torch.tensor([0, 40], **i32), 40)
    ref = _exact(model, torch.cat([_ids(3, 2), ids[1:41]]))[0].detach()[3:]
    plain = _off(_plain(model, torch.cat([_ids(3, 2), ids[1:41]]))[3:].detach(), ref)
    assert _off(again, ref) <= 1.5 * plain
    check_errors()


def test_logits_of_a_sequence_without_room_are_nan():
    """It stays as it was, and what its rows hold cannot be taken for an answer."""
    from multi_gpu_flashattention_b200 import KernelStatusError
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    model = _model(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = model.make_cache(pages=3, page_size=16, slots=4, max_tokens=64)
    ids, cu, most = _batch([_ids(5, 1), _ids(33, 2), _ids(7, 3), _ids(7, 4)])
    tail = torch.cat([ids, _ids(3, 5)])  # rows of no sequence
    # 1 page, 3 pages of the 2 left, a slot out of range, a slot named again
    out = model.serve(tail, cache, torch.tensor([2, 0, 4, 2], **i32), cu, most)
    with pytest.raises(KernelStatusError):
        check_errors()
    assert cache.lens.tolist() == [0, 0, 5, 0]
    assert torch.isfinite(out[:5]).all() and out[5:52].isnan().all()
    out = model.serve(ids[:5], cache, torch.tensor([2], **i32), torch.tensor([0, 5], **i32), 5)
    assert torch.isfinite(out).all()
    check_errors()


def test_the_plain_model_computes_the_plain_formulas():
    """Without fused_ops, to the bit: norms and rotary positions in torch, attention as
    ring_attention gives it; with it, other roundings of the same values."""
    from multi_gpu_flashattention_b200 import RingLayout, ring_attention
    model, ids = _model(torch.bfloat16), _ids(200, 9)
    lay = RingLayout("contiguous", 200, 1, mask="causal")
    norm = lambda x, w: (x.float() * torch.rsqrt(x.float().pow(2).mean(-1, keepdim=True) + 1e-6)).to(x.dtype) * w
    inv = 10000.0 ** (-torch.arange(0, D // 2, device="cuda", dtype=torch.float32) * 2 / D)
    ang = torch.arange(200, device="cuda", dtype=torch.float32)[:, None] * inv

    def rot(t):
        a, b = t[..., :D // 2].float(), t[..., D // 2:].float()
        c, s = ang.cos()[None, :, None], ang.sin()[None, :, None]
        return torch.cat([a * c - b * s, a * s + b * c], -1).to(t.dtype)

    with torch.no_grad():
        x = model.embed(ids[None])
        for blk in model.blocks:
            h = norm(x, blk.norm1.weight)
            q, k, v = (w(h).view(1, 200, -1, D) for w in (blk.wq, blk.wk, blk.wv))
            a = ring_attention(rot(q), rot(k), v.contiguous(), causal=True, layout=lay)
            x = x + blk.wo(a.reshape(1, 200, -1))
            h = norm(x, blk.norm2.weight)
            x = x + blk.w2(F.silu(blk.w1(h)) * blk.w3(h))
        want = model.head(norm(x, model.norm.weight))
        plain = model(ids[None], lay)
        assert torch.equal(plain, want)
        for m in [model, *model.blocks]:
            m.fused_ops = True
        fused = model(ids[None], lay)
        assert not torch.equal(fused, plain)
        ref = _exact(model, ids)[0]
        assert _off(fused[0], ref) <= 1.5 * _off(plain[0], ref)
        for m in [model, *model.blocks]:
            m.fused_ops = False
        assert torch.equal(model(ids[None], lay), want)


def test_serving_steps_in_a_graph():
    """A decode step captured once and replayed, a sequence running out of pages on the way:
    the same logits and the same cache as step by step, NaN from the refused step on."""
    from multi_gpu_flashattention_b200 import KernelStatusError
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    model = _model(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device="cuda")
    slots, cu = torch.tensor([2, 0], **i32), torch.tensor([0, 1, 2], **i32)
    first, cu1, most1 = _batch([_ids(14, 1), _ids(3, 2)])
    runs = []
    for graphed in (False, True):
        cache = model.make_cache(pages=3, page_size=16, slots=3, max_tokens=64)  # one page to spare
        model.serve(first, cache, slots, cu1, most1)
        ids, got = _ids(2, 3), []
        if graphed:
            saved = [t.clone() for t in (cache.page_table, cache.lens, cache.refs, cache.grown)]
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                model.serve(ids, cache, slots, cu, 1)
                for t, u in zip((cache.page_table, cache.lens, cache.refs, cache.grown), saved):
                    t.copy_(u)
            torch.cuda.current_stream().wait_stream(s)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = model.serve(ids, cache, slots, cu, 1)
        for i in range(20):  # sequence 2 grows into the last page, sequence 0 stays at 16 tokens
            ids.copy_(_ids(2, 10 + i))
            if graphed:
                graph.replay()
            else:
                try:
                    out = model.serve(ids, cache, slots, cu, 1)
                except KernelStatusError:
                    out = model.serve(ids, cache, slots, cu, 1)
            got.append(out.clone())
        with pytest.raises(KernelStatusError, match="too few free pages"):
            check_errors()
        assert cache.lens.tolist() == [16, 0, 32]
        runs.append(torch.stack(got))
    bad = runs[0].isnan().all(-1)
    assert torch.equal(bad, runs[1].isnan().all(-1))
    assert bad[:, 0].tolist() == [False] * 18 + [True] * 2 and bad[:, 1].tolist() == [False] * 13 + [True] * 7
    assert torch.equal(runs[0].nan_to_num(), runs[1].nan_to_num())
    check_errors()
