"""PagedKVCache.append against the definition in 64 bits: the queries returned, the keys and
values in their pages, everything else left as it was. Tolerances as in
test_norm_rotary_gpu.py; without the norm a value is off by u|y| + 1e-6 (|a| + |b|)
magnitude (test_rotary_gpu.py), and columns that are not rotated, and the values, are
copies."""
import pytest
import torch

from test_norm_rotary_gpu import angle_error, close, reference

pytestmark = pytest.mark.gpu


def _cache(pages=40, page=16, heads=2, D=64, slots=8, layers=2, dtype=torch.bfloat16, max_tokens=320):
    from multi_gpu_flashattention_b200 import PagedKVCache
    c = PagedKVCache.allocate(layers, pages, page, heads, D, slots, max_tokens, dtype=dtype)
    c.k.fill_(7.0)
    c.v.fill_(-7.0)
    return c


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _batch(T, H, Hk, D, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    qkv = torch.randn(T, H + 2 * Hk, D, device="cuda", generator=g).to(dtype)
    return qkv.split([H, Hk, Hk], 1)


def _check(cache, before, layer, q, k, v, out, pos, inv, slots, cu, ws, interleaved, magnitude, grew=None):
    """Rows of sequences in `grew` (default: all) are in their pages, all others are not."""
    T, rd = q.shape[0], 2 * inv.numel()
    ref = []
    for x, w in ((q, ws and ws[0]), (k, ws and ws[1])):
        if ws:
            r = reference(x[None], w, x[None], pos[None], inv, 1e-6, interleaved, magnitude)
            ref.append((r["y"][0], r["y_size"][0], 2e-6))
        else:
            one = torch.ones(x.shape[-1], device="cuda")
            r = reference(x[None], one, x[None], pos[None], inv, 1e-6, interleaved, magnitude)
            scale = (x.double().pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
            ref.append((r["y"][0] * scale, r["y_size"][0] * scale, 1e-6))
    more = angle_error(pos, inv)
    close(out, ref[0][0], ref[0][1], ref[0][2] + more)
    if not ws:
        assert torch.equal(out[..., rd:], q[..., rd:])
    want_k, want_v = before[0].clone(), before[1].clone()
    table, lens, p = cache.page_table.tolist(), cache.lens.tolist(), cache.page_size
    cu = cu.tolist()
    written = torch.zeros(cache.k.shape[:3], dtype=torch.bool, device="cuda")
    for b, slot in enumerate(slots.tolist()):
        if grew is not None and b not in grew:
            continue
        n = cu[b + 1] - cu[b]
        for i in range(n):
            at = lens[slot] - n + i
            cell = (layer, table[slot][at // p], at % p)
            row = cu[b] + i
            close(cache.k[cell], ref[1][0][row], ref[1][1][row], ref[1][2] + more)
            if not ws:
                assert torch.equal(cache.k[cell][..., rd:], k[row][..., rd:])
            assert torch.equal(cache.v[cell], v[row])
            written[cell] = True
    assert torch.equal(cache.k[~written], want_k[~written]) and torch.equal(cache.v[~written], want_v[~written])


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hk,D,rd,page,interleaved", [(4, 2, 64, 64, 16, False), (3, 1, 128, 128, 32, False),
                                                       (8, 8, 64, 24, 16, False), (4, 2, 128, 50, 64, False),
                                                       (4, 2, 64, 32, 16, True), (40, 1, 128, 128, 16, False),
                                                       (2, 2, 128, 96, 16, True)])
def test_against_the_definition(H, Hk, D, rd, page, interleaved, dtype, norm):
    from multi_gpu_flashattention_b200 import rotary_frequencies
    inv, mag = rotary_frequencies(rd, scaling="ramp", factor=2.0, original_length=64, device="cuda")
    cache = _cache(page=page, heads=Hk, D=D, dtype=dtype)
    ws = [(1 + 0.2 * torch.randn(D, device="cuda")).to(torch.float32 if rd % 3 else dtype) for _ in range(2)] if norm else None
    slots = _ints([5, 0, 3])
    for step, lens in enumerate(([19, 1, 33], [1, 1, 1], [0, 40, 2])):
        cu = _ints([0, lens[0], lens[0] + lens[1], sum(lens)])
        T = sum(lens)
        q, k, v = _batch(T, H, Hk, D, dtype, seed=step)
        pos = cache.reserve(slots, cu, T)
        before = cache.k.clone(), cache.v.clone()
        layer = step % 2
        more = dict(q_weight=ws[0], k_weight=ws[1]) if norm else {}
        out = cache.append(layer, q, k, v, pos, inv, slots, cu, interleaved=interleaved, magnitude=mag, **more)
        _check(cache, before, layer, q, k, v, out, pos, inv, slots, cu, ws, interleaved, mag)


def test_rows_outside_and_refused_sequences():
    """A batch padded for a graph; a slot named twice; one that got no pages; one out of range."""
    from multi_gpu_flashattention_b200 import KernelStatusError, rotary_frequencies
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    inv, _ = rotary_frequencies(64, device="cuda")
    cache = _cache(pages=6)
    slots, cu = _ints([1, 2, 1, 3, 99]), _ints([2, 22, 25, 28, 200, 201])
    T = 210
    q, k, v = _batch(T, 4, 2, 64, torch.bfloat16, 3)
    pos = cache.reserve(slots, cu, T)  # slot 1: 2 pages, slot 2: 1; again 1: refused; 3: 11 pages, refused
    before = cache.k.clone(), cache.v.clone()
    out = cache.append(0, q, k, v, pos, inv, slots, cu)
    _check(cache, before, 0, q, k, v, out, pos, inv, slots, cu, None, False, 1.0, grew={0, 1})
    with pytest.raises(KernelStatusError):
        check_errors()


def test_together_with_attention_and_write():
    """Without weights append() is apply_rotary() and write(), to the bit, and attend() reads it."""
    from multi_gpu_flashattention_b200 import apply_rotary, rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    cache = _cache()
    slots, cu = _ints([2, 4]), _ints([0, 30, 47])
    q, k, v = _batch(47, 4, 2, 64, torch.bfloat16, 5)
    pos = cache.reserve(slots, cu, 47)
    a = cache.append(0, q, k, v, pos, inv, slots, cu)
    b, kr = apply_rotary(q, k, pos, inv)
    cache.write(1, kr, v, slots, cu)
    assert torch.equal(a, b) and torch.equal(cache.k[0], cache.k[1]) and torch.equal(cache.v[0], cache.v[1])
    assert torch.isfinite(cache.attend(0, a, slots, cu, 30)).all()


def test_empty_batches_positions_and_streams():
    from multi_gpu_flashattention_b200 import rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    cache = _cache()
    q, k, v = _batch(0, 4, 2, 64, torch.bfloat16)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert cache.append(0, q, k, v, none, inv, _ints([]), _ints([0])).shape == (0, 4, 64)
    q, k, v = _batch(5, 4, 2, 64, torch.bfloat16)
    before = cache.k.clone()
    # rows without a sequence: queries are rotated, nothing is written
    out = cache.append(0, q, k, v, torch.zeros(5, dtype=torch.int64, device="cuda"), inv, _ints([]), _ints([0]))
    assert torch.equal(out, q) and torch.equal(cache.k, before)
    side = torch.cuda.Stream()
    slots, cu = _ints([0]), _ints([0, 5])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pos = cache.reserve(slots, cu, 5)
        before = cache.k.clone(), cache.v.clone()
        out = cache.append(1, q, k, v, pos.long() + 100000, inv, slots, cu)
    side.synchronize()
    _check(cache, before, 1, q, k, v, out, pos.long() + 100000, inv, slots, cu, None, False, 1.0)


def test_captured_step():
    from multi_gpu_flashattention_b200 import rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    caches = [_cache(), _cache()]
    slots, cu = _ints([3, 1]), _ints([0, 1, 2])
    q, k, v = (t.contiguous() for t in _batch(2, 4, 2, 64, torch.bfloat16))
    w = torch.ones(64, device="cuda")

    def step(c):
        pos = c.reserve(slots, cu, 2)
        return c.append(0, q, k, v, pos, inv, slots, cu, q_weight=w, k_weight=w)

    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        got = step(caches[0])
    for i in range(20):
        nq, nk, nv = _batch(2, 4, 2, 64, torch.bfloat16, seed=i)
        q.copy_(nq), k.copy_(nk), v.copy_(nv)
        graph.replay()
        want = step(caches[1])
        assert torch.equal(got, want)
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
    assert caches[0].lens.tolist()[3] == 20


def test_refusals():
    from multi_gpu_flashattention_b200 import rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    cache = _cache()
    q, k, v = _batch(2, 4, 2, 64, torch.bfloat16)
    slots, cu = _ints([0]), _ints([0, 2])
    pos = cache.reserve(slots, cu, 2)
    w = torch.ones(64, device="cuda")
    ok = dict(layer=0, q=q, k=k, v=v, positions=pos, inv_freq=inv, slots=slots, cu_seqlens=cu)

    def refused(match, **change):
        with pytest.raises(RuntimeError, match=match):
            cache.append(**{**ok, **change})

    cache.append(**ok)
    refused("is not one of the cache's", layer=2)
    refused("is not one of the cache's", layer=-1)
    refused("come together", q_weight=w)
    refused("cache's dtype", v=v.half())
    refused("must be \\[tokens, kv_heads, head_dim\\]", k=q, v=q)
    refused("with new_k's tokens", q=q[:1])
    refused("positions must be", positions=pos[:1])
    refused("sequences \\+ 1", cu_seqlens=_ints([0, 1, 2]))
    refused("contiguous head_dim", q=torch.zeros(2, 64, 4, device="cuda", dtype=torch.bfloat16).transpose(1, 2))
    refused("no gradient", q=q.clone().requires_grad_())
    refused("head_dim", q_weight=w[:32], k_weight=w[:32])


def test_strides_of_single_rows_mean_nothing():
    """One token and one head, cut from rows of an odd length."""
    from multi_gpu_flashattention_b200 import apply_norm_rotary, apply_rotary, rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    w = torch.ones(64, device="cuda")
    cache = _cache(heads=1)
    wide = torch.randn(3, 1, 1, 67, device="cuda").bfloat16()
    q, k, v = (wide[i, :, :, :64].as_strided((1, 1, 64), (67, 67, 1), 0) for i in range(3))
    q, k, v = (torch.empty_strided((1, 1, 64), (67, 5, 1), dtype=torch.bfloat16, device="cuda").copy_(t) for t in (q, k, v))
    pos = cache.reserve([0], [0, 1], 1)
    before = cache.k.clone(), cache.v.clone()
    out = cache.append(0, q, k, v, pos + 9, inv, _ints([0]), _ints([0, 1]))
    _check(cache, before, 0, q, k, v, out, pos + 9, inv, _ints([0]), _ints([0, 1]), None, False, 1.0)
    assert torch.equal(apply_rotary(q, None, pos + 9, inv), out)
    assert torch.equal(apply_norm_rotary(q, None, pos + 9, inv, w, None), apply_norm_rotary(q.contiguous(), None, pos + 9, inv, w, None))


def test_large_pool_offsets():
    """Pages that begin beyond 2^31 elements of the pool."""
    from multi_gpu_flashattention_b200 import PagedKVCache, rotary_frequencies
    inv, _ = rotary_frequencies(128, device="cuda")
    pages = (1 << 31) // (64 * 8 * 128) + 3
    c = PagedKVCache.allocate(1, pages, 64, 8, 128, 2, 128)
    c.refs[:pages - 2] = 1  # the last two are free
    q, k, v = _batch(70, 16, 8, 128, torch.bfloat16)
    slots, cu = _ints([1]), _ints([0, 70])
    pos = c.reserve(slots, cu, 70)
    out = c.append(0, q, k, v, pos, inv, slots, cu)
    assert c.page_table[1].tolist() == [pages - 2, pages - 1]
    one = torch.ones(128, device="cuda")
    for x, got in ((q, out), (k, c.k[0, -2:].flatten(0, 1)[:70])):
        r = reference(x[None], one, x[None], pos[None], inv, 1e-6, False, 1.0)
        scale = (x.double().pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        close(got, r["y"][0] * scale, r["y_size"][0] * scale, 1e-6)
    assert torch.equal(c.v[0, -2:].flatten(0, 1)[:70], v)
