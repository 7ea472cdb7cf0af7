"""The operators around attention in a decoder layer, measured over the range in which they are used.

    norm       root-mean-square norm with the residual's addition: a training step
               (forward and gradients), or the serving form with an output in 8 bits
               and its scales
    rotary     rotary positions on queries and keys: a training step, or serving
    attention  a chunk of new tokens (or one) of each sequence of a batch against a
               paged cache of keys and values
    pages      the cache's pages: room for new tokens and their keys and values
               written, sequences freed and forked, the pool compacted

`run` computes each in its plain form (elementary torch operations in 32 bits), or,
where `own` is true, calls the package's operators. `exact` gives the same outputs in
64 bits.
"""
import math

import torch

own = False

BF16, FP16, FP32 = "bfloat16", "float16", "float32"
E4M3_MAX = 448.0


# ------------------------------------------------------------------------- cases
def listed():
    return [
        # One layer's norm in training: 16384 tokens of width 4096 (32 heads of 128).
        dict(name="norm train 16384x4096", op="norm", mode="train", rows=16384, dim=4096,
             dtype=BF16, residual=True, group=0),
        # An odd number of tokens of an odd width in fp32, without a residual.
        dict(name="norm train 1537x1000 fp32", op="norm", mode="train", rows=1537, dim=1000,
             dtype=FP32, residual=False, group=0),
        # Serving: eight decoding sequences, 8-bit output with a scale for each 128 columns.
        dict(name="norm 8-bit 8x4096", op="norm", mode="serve8", rows=8, dim=4096, dtype=BF16,
             residual=True, group=128),
        # One layer's positions in training: 32768 tokens, 32 query and 8 key heads, extended
        # context (interpolation by frequency).
        dict(name="rotary train 32768 tokens", op="rotary", mode="train", tokens=32768, heads=32,
             kv_heads=8, head_dim=128, rotary_dim=128, interleaved=False, scaling="ramp",
             start=98304, dtype=BF16),
        # Serving: 61 decoding tokens far into their contexts, interleaved pairs, half the head.
        dict(name="rotary serve 61 tokens", op="rotary", mode="serve", tokens=61, heads=32,
             kv_heads=8, head_dim=128, rotary_dim=64, interleaved=True, scaling="none",
             start=131071, dtype=FP16),
        # Decoding, small model and short contexts: latency.
        dict(name="decode 4 short", op="attention", seqs=4, new=1, ragged_new=False, kv_max=512,
             kv_min=33, heads=8, kv_heads=2, head_dim=64, page=16, dtype=FP16),
        # Decoding, one sequence of the longest context.
        dict(name="decode 1 of 131072", op="attention", seqs=1, new=1, ragged_new=False,
             kv_max=131072, kv_min=131071, heads=32, kv_heads=8, head_dim=128, page=64, dtype=BF16),
        # Decoding, a full batch with ragged contexts.
        dict(name="decode 64 ragged", op="attention", seqs=64, new=1, ragged_new=False, kv_max=8192,
             kv_min=1, heads=32, kv_heads=8, head_dim=128, page=16, dtype=BF16),
        # Chunked prefill of a few sequences with ragged chunks and histories.
        dict(name="chunk 5 ragged x512", op="attention", seqs=5, new=512, ragged_new=True,
             kv_max=16384, kv_min=600, heads=32, kv_heads=8, head_dim=128, page=32, dtype=BF16),
        # One large chunk over a long history.
        dict(name="chunk 2048 of 32768", op="attention", seqs=1, new=2048, ragged_new=False,
             kv_max=32768, kv_min=32700, heads=32, kv_heads=8, head_dim=128, page=64, dtype=BF16),
        # A serving step's room and writes: ragged chunks of 16 sequences into one layer's pages.
        dict(name="pages append 16x256", op="pages", mode="append", layers=1, pages=2048, page=64,
             seqs=16, held=60, new=256, kv_heads=8, head_dim=128, dtype=BF16),
        # A third of the sequences leave, then the pool is compacted.
        dict(name="pages compact 2048", op="pages", mode="compact", layers=2, pages=2048, page=64,
             seqs=48, held=40, new=0, kv_heads=8, head_dim=128, dtype=BF16),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "rotary", "attention", "attention", "attention", "pages"])
    if op == "norm":
        mode = rng.choice(["train", "serve8"])
        group = rng.choice([0, 64, 128]) if mode == "serve8" else 0
        dim = group * _log(rng, 1, 64) if group else _log(rng, 32, 8192)
        rows = _log(rng, 1, min(16384, 16384 * 4096 // dim))
        return dict(op=op, mode=mode, rows=rows, dim=dim, group=group,
                    dtype=rng.choice([BF16, FP16] if mode == "serve8" else [BF16, FP16, FP32]),
                    residual=rng.random() < 0.7)
    if op == "rotary":
        head_dim = rng.choice([64, 128])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4])
        return dict(op=op, mode=rng.choice(["train", "serve"]), heads=heads, kv_heads=kv,
                    tokens=_log(rng, 1, 32768 * 32 // max(32, heads)), head_dim=head_dim,
                    rotary_dim=rng.choice([head_dim, head_dim // 2, 2 * rng.randint(1, head_dim // 2)]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ramp"]),
                    start=_log(rng, 1, 1 << 20), dtype=rng.choice([BF16, FP16, FP32]))
    if op == "attention":
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
        new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 2048)])
        seqs = _log(rng, 1, 64 if new <= 16 else 8)
        # history such that scores and pages of a pass stay below the largest listed ones
        most = min(131072, (2048 * 32768 * 32) // (seqs * new * heads), (64 * 8192 * 8) // (seqs * kv))
        kv_max = max(new, _log(rng, max(new, 16), max(new, most, 16)))
        return dict(op=op, seqs=seqs, new=new, ragged_new=new > 1 and rng.random() < 0.7,
                    kv_max=kv_max, kv_min=rng.randint(new, kv_max), heads=heads, kv_heads=kv,
                    head_dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice([BF16, FP16]))
    mode = rng.choice(["append", "fork", "compact"])
    page = rng.choice([16, 32, 64])
    seqs = _log(rng, 3, 48)
    held = _log(rng, 1, 40)
    new = _log(rng, 1, 4 * page) if mode == "append" else 0
    most = seqs * (held + 4 + new // page) + 8
    return dict(op=op, mode=mode, layers=1 if mode == "append" else rng.choice([1, 2]), page=page,
                pages=int(most * rng.uniform(1.0, 1.3)), seqs=seqs, held=held, new=new,
                kv_heads=rng.choice([2, 8]), head_dim=rng.choice([64, 128]),
                dtype=rng.choice([BF16, FP16]))


# ------------------------------------------------------------------------- inputs
def _dtype(case):
    return getattr(torch, case["dtype"])


def _rng(seed):
    """A generator on the host (sizes, places) and one on the device (values)."""
    return torch.Generator().manual_seed(seed), torch.Generator("cuda").manual_seed(seed)


def _randn(shape, dtype, gen, std=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(0.0, std, generator=gen)


def _frequencies(case):
    """Angles a position (radians) of each rotated pair, in 64 bits, and the factor on the
    rotated values. "linear" divides every frequency by 4. "ramp" interpolates by frequency:
    pairs that turn more than 32 times in the original 32768 positions keep theirs, those
    that turn less than once are divided by 4, with a linear ramp between, and the values
    grow by 0.1 ln 4 + 1."""
    rd, base, factor, original = case["rotary_dim"], 10000.0, 4.0, 32768
    inv = base ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    if case["scaling"] == "linear":
        return inv / factor, 1.0
    if case["scaling"] == "ramp":
        def pair_of(turns):
            return rd * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo = max(math.floor(pair_of(32.0)), 0)
        hi = min(math.ceil(pair_of(1.0)), rd - 1)
        ramp = ((torch.arange(rd // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return inv * (1 - ramp) + inv / factor * ramp, 0.1 * math.log(factor) + 1.0
    return inv, 1.0


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _chunks(case):
    """Ragged numbers of new tokens: the same for every seed, since they give the outputs' shapes."""
    host = torch.Generator().manual_seed(case["seqs"])
    return [case["new"]] + torch.randint(1, case["new"] + 1, (case["seqs"] - 1,), generator=host).tolist()


def prepare(case, seed):
    return {"norm": _prepare_norm, "rotary": _prepare_rotary, "attention": _prepare_attention,
            "pages": _prepare_pages}[case["op"]](case, seed)


def _prepare_norm(case, seed):
    _, gen = _rng(seed)
    dt, shape = _dtype(case), (case["rows"], case["dim"])
    train = case["mode"] == "train"
    s = dict(case=case, eps=1e-6, x=_randn(shape, dt, gen).requires_grad_(train),
             w=(1 + 0.1 * torch.randn(case["dim"], device="cuda", generator=gen)).to(dt).requires_grad_(train))
    s["r"] = _randn(shape, dt, gen, 2.0).requires_grad_(train) if case["residual"] else None
    if train:
        s["dy"] = _randn(shape, dt, gen)
        s["dh"] = _randn(shape, dt, gen) if case["residual"] else None
    return s


def _prepare_rotary(case, seed):
    host, gen = _rng(seed)
    dt, t = _dtype(case), case["tokens"]
    train = case["mode"] == "train"
    inv, magnitude = _frequencies(case)
    pos = torch.arange(t) + case["start"] if train else \
        torch.randint(0, case["start"] + 1, (t,), generator=host)
    s = dict(case=case, inv=inv.cuda(), magnitude=magnitude, pos=pos.cuda(),
             q=_randn((t, case["heads"], case["head_dim"]), dt, gen).requires_grad_(train),
             k=_randn((t, case["kv_heads"], case["head_dim"]), dt, gen).requires_grad_(train))
    if train:
        s["dq"], s["dk"] = _randn(s["q"].shape, dt, gen), _randn(s["k"].shape, dt, gen)
    return s


def _prepare_attention(case, seed):
    host, gen = _rng(seed)
    dt, n, p = _dtype(case), case["seqs"], case["page"]
    new = _chunks(case) if case["ragged_new"] else [case["new"]] * n
    kv = [int(torch.randint(case["kv_min"], case["kv_max"] + 1, (1,), generator=host)) for _ in range(n)]
    kv[0] = case["kv_max"]
    kv = [max(a, b) for a, b in zip(kv, new)]
    need = [-(-a // p) for a in kv]
    width, pool = -(-case["kv_max"] // p), sum(need)
    order = torch.randperm(pool, generator=host).tolist()
    table, at = [], 0
    for k in need:
        table.append(order[at:at + k] + [-1] * (width - k))
        at += k
    cu = [0]
    for a in new:
        cu.append(cu[-1] + a)
    shape = (pool, p, case["kv_heads"], case["head_dim"])
    return dict(case=case, q=_randn((cu[-1], case["heads"], case["head_dim"]), dt, gen),
                k=_randn(shape, dt, gen), v=_randn(shape, dt, gen), table=_ints(table),
                lens=_ints(kv), cu=_ints(cu), max_new=max(new))


def _prepare_pages(case, seed):
    """A pool in the middle of its life: the sequences' pages lie anywhere in it. `meta` is
    what the steps change: the table, the lengths, how many sequences hold each page, and
    how far each sequence grew last."""
    host, gen = _rng(seed)
    dt, n, p, pages = _dtype(case), case["seqs"], case["page"], case["pages"]
    held = [int(torch.randint(max(1, case["held"] // 2), case["held"] + 1, (1,), generator=host)) for _ in range(n)]
    lens = [(h - 1) * p + int(torch.randint(1, p + 1, (1,), generator=host)) for h in held]
    slots = 2 * n
    width = case["held"] + 2 + -(-case["new"] // p)
    order = torch.randperm(pages, generator=host)
    table, refs, at = torch.full((slots, width), -1, dtype=torch.int32), torch.zeros(pages, dtype=torch.int32), 0
    where = torch.randperm(slots, generator=host).tolist()
    busy, idle = where[:n], where[n:]
    length = torch.zeros(slots, dtype=torch.int32)
    for i, slot in enumerate(busy):
        table[slot, :held[i]] = order[at:at + held[i]].int()
        refs[order[at:at + held[i]]] = 1
        at += held[i]
        length[slot] = lens[i]
    meta = torch.cat([table.flatten(), length, refs, torch.zeros(slots, dtype=torch.int32)]).cuda()
    shape = (case["layers"], pages, p, case["kv_heads"], case["head_dim"])
    s = dict(case=case, k=_randn(shape, dt, gen), v=_randn(shape, dt, gen), meta=meta.clone(), kept=meta)
    cuts = [slots * width, slots, pages, slots]
    table, length, refs, grown = s["meta"].split(cuts)
    s.update(table=table.view(slots, width), lens=length, refs=refs, grown=grown)
    if case["mode"] == "append":
        new = _chunks(case)
        cu = [0]
        for a in new:
            cu.append(cu[-1] + a)
        s.update(slots=_ints(busy), cu=_ints(cu), most=case["new"],
                 new_k=_randn((cu[-1],) + shape[3:], dt, gen), new_v=_randn((cu[-1],) + shape[3:], dt, gen))
    else:
        leave = n // 3
        s["leave"] = _ints(busy[:leave])
        stay = busy[leave:]
        if case["mode"] == "fork":
            s["src"], s["dst"] = _ints(stay), _ints(idle[:len(stay)])
    return s


# ------------------------------------------------------------------------- one pass
def run(s):
    return {"norm": _run_norm, "rotary": _run_rotary, "attention": _run_attention,
            "pages": _run_pages}[s["case"]["op"]](s)


def _run_norm(s):
    c = s["case"]
    if own:
        from multi_gpu_flashattention_b200 import rms_norm, rms_norm_fp8
        if c["mode"] == "serve8":
            out = rms_norm_fp8(s["x"], s["w"], residual=s["r"], eps=s["eps"], group=c["group"])
            return _eight(*out)
        if c["residual"]:
            y, h = rms_norm(s["x"], s["w"], residual=s["r"], eps=s["eps"])
            dx, dr, dw = torch.autograd.grad([y, h], [s["x"], s["r"], s["w"]], [s["dy"], s["dh"]])
            return dict(y=y, h=h, dx=dx, dr=dr, dw=dw)
        y = rms_norm(s["x"], s["w"], eps=s["eps"])
        dx, dw = torch.autograd.grad([y], [s["x"], s["w"]], [s["dy"]])
        return dict(y=y, dx=dx, dw=dw)
    with torch.no_grad():
        dt = s["x"].dtype
        # the new residual stream is an output: it is rounded to its type, and the norm reads it
        h = s["x"].float() + s["r"].float() if c["residual"] else s["x"].float()
        h = h.to(dt)
        hf, w = h.float(), s["w"].float()
        rstd = torch.rsqrt(hf.square().mean(-1, keepdim=True) + s["eps"])
        n = hf * rstd
        y = n * w
        if c["mode"] == "serve8":
            g = c["group"] or c["dim"]
            yg = y.view(c["rows"], -1, g)
            scale = yg.abs().amax(-1) / E4M3_MAX
            scale = torch.where(scale > 0, scale, torch.ones_like(scale))
            y8 = (yg / scale[..., None]).to(torch.float8_e4m3fn).view(c["rows"], c["dim"])
            return _eight(y8, scale, h if c["residual"] else None)
        dy = s["dy"].float()
        dw = (dy * n).sum(0)
        wdy = dy * w
        dx = rstd * (wdy - n * (wdy * n).mean(-1, keepdim=True))
        if c["residual"]:
            dx = (dx + s["dh"].float()).to(dt)
            return dict(y=y.to(dt), h=h, dx=dx, dr=dx, dw=dw.to(dt))
        return dict(y=y.to(dt), dx=dx.to(dt), dw=dw.to(dt))


def _eight(y8, scale, h=None):
    """The values that the 8-bit output stands for, the scales, and the new residual stream."""
    rows, dim = y8.shape
    y = (y8.float().view(rows, scale.shape[-1], -1) * scale[..., None]).view(rows, dim)
    out = dict(y=y.to(torch.bfloat16), scale=scale)
    return out if h is None else dict(out, h=h)


def _rotate(x, cos, sin, rotary_dim, interleaved):
    xf = x[..., :rotary_dim].to(cos.dtype)
    if interleaved:
        a, b = xf[..., 0::2], xf[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = xf[..., :rotary_dim // 2], xf[..., rotary_dim // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y.to(x.dtype), x[..., rotary_dim:]], -1) if cos.dtype == torch.float32 else \
        torch.cat([y, x[..., rotary_dim:].to(cos.dtype)], -1)


def _run_rotary(s):
    c = s["case"]
    if own:
        from multi_gpu_flashattention_b200 import apply_rotary
        q, k = apply_rotary(s["q"], s["k"], s["pos"], s["inv"], interleaved=c["interleaved"],
                            magnitude=s["magnitude"])
        if c["mode"] == "serve":
            return dict(q=q, k=k)
        dq, dk = torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])
        return dict(q=q, k=k, dq=dq, dk=dk)
    with torch.no_grad():
        angle = s["pos"].double()[:, None] * s["inv"]  # far positions: 64 bits
        cos = (angle.cos() * s["magnitude"]).float()[:, None, :]
        sin = (angle.sin() * s["magnitude"]).float()[:, None, :]
        rd, il = c["rotary_dim"], c["interleaved"]
        out = dict(q=_rotate(s["q"], cos, sin, rd, il), k=_rotate(s["k"], cos, sin, rd, il))
        if c["mode"] == "train":  # the transpose of a rotation is the rotation back
            out.update(dq=_rotate(s["dq"], cos, -sin, rd, il), dk=_rotate(s["dk"], cos, -sin, rd, il))
        return out


def _run_attention(s):
    c = s["case"]
    if own:
        from multi_gpu_flashattention_b200 import paged_attention
        out, lse = paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"],
                                   s["max_new"], return_lse=True)
        return dict(out=out, lse=lse)
    q, m, p = s["q"], s["max_new"], c["page"]
    t, hq, d = q.shape
    hkv, b = c["kv_heads"], c["seqs"]
    g = hq // hkv
    dev = q.device
    pages = s["table"].long().clamp(min=0)
    cu, lens = s["cu"].long(), s["lens"].long()
    keys = pages.shape[1] * p
    k = s["k"][pages].view(b, keys, hkv, d).permute(0, 2, 1, 3).float()
    v = s["v"][pages].view(b, keys, hkv, d).permute(0, 2, 1, 3).float()
    row = cu[:-1, None] + torch.arange(m, device=dev)
    qp = q[row.clamp(max=t - 1)].float().view(b, m, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, m * g, d)
    scores = (qp @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).view(b, hkv, m, g, keys)
    n_new = cu[1:] - cu[:-1]
    last = lens[:, None] - n_new[:, None] + torch.arange(m, device=dev)  # a token sees itself and all before
    hidden = torch.arange(keys, device=dev) > last[:, :, None]
    scores.masked_fill_(hidden[:, None, :, None, :], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    e = scores.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.view(b, hkv, m * g, keys) @ v).view(b, hkv, m, g, d) / total.clamp(min=1e-30)
    lse = (top + total.log()).squeeze(-1)
    # back to packed rows
    at = torch.arange(t, device=dev)
    seq = torch.searchsorted(cu, at, right=True) - 1
    i = at - cu[seq]
    out = o.permute(0, 2, 1, 3, 4)[seq, i].reshape(t, hq, d)
    return dict(out=out.to(q.dtype), lse=lse.permute(0, 2, 1, 3)[seq, i].reshape(t, hq).t().contiguous())


def _run_pages(s):
    c = s["case"]
    s["meta"].copy_(s["kept"])  # the same step again
    if own:
        cache = s.get("cache")
        if cache is None:
            from multi_gpu_flashattention_b200 import PagedKVCache
            cache = s["cache"] = PagedKVCache(s["k"], s["v"], s["table"], s["lens"], s["refs"], s["grown"])
        if c["mode"] == "append":
            pos = cache.reserve(s["slots"], s["cu"], s["new_k"].shape[0])
            cache.write(0, s["new_k"], s["new_v"], s["slots"], s["cu"])
            return _pages_out(s, positions=pos)
        cache.free(s["leave"])
        if c["mode"] == "fork":
            cache.fork(s["src"], s["dst"])
        else:
            cache.compact()
        return _pages_out(s)
    table, lens, refs, grown, p = s["table"], s["lens"], s["refs"], s["grown"], c["page"]
    if c["mode"] == "append":
        slots, cu = s["slots"].long(), s["cu"].long()
        n_new = cu[1:] - cu[:-1]
        old = lens[slots].long()
        _take(table, refs, slots, (old + p - 1) // p, (old + n_new + p - 1) // p, s["most"] // p + 1)
        lens[slots] = (old + n_new).int()
        grown[slots] = n_new.int()
        at = torch.arange(s["new_k"].shape[0], device=cu.device)
        seq = torch.searchsorted(cu, at, right=True) - 1
        pos = old[seq] + at - cu[seq]
        cell = table[slots[seq], pos // p].long() * p + pos % p
        s["k"][0].view(-1, *s["k"].shape[3:]).index_copy_(0, cell, s["new_k"])
        s["v"][0].view(-1, *s["v"].shape[3:]).index_copy_(0, cell, s["new_v"])
        return _pages_out(s, positions=pos.int())
    gone = s["leave"].long()
    theirs = table[gone]
    refs.index_add_(0, theirs.clamp(min=0).flatten().long(), -(theirs >= 0).flatten().int())
    table[gone] = -1
    lens[gone] = 0
    grown[gone] = 0
    if c["mode"] == "fork":
        src, dst = s["src"].long(), s["dst"].long()
        length = lens[src].long()
        whole, part = length // p, length % p
        row = torch.where(torch.arange(table.shape[1], device=table.device) < whole[:, None], table[src], -1)
        refs.index_add_(0, row.clamp(min=0).flatten().long(), (row >= 0).flatten().int())
        table[dst] = row
        lens[dst] = lens[src]
        grown[dst] = 0
        _take(table, refs, dst, whole, whole + (part > 0), 1)
        # the tokens of the last page, where it is not full, get a page of their own
        cols = torch.arange(p, device=table.device)
        has = cols < part[:, None]
        last = whole.clamp(max=table.shape[1] - 1)[:, None]
        a = (table[src[:, None], last].long().clamp(min=0) * p + cols)[has]
        b = (table[dst[:, None], last].long().clamp(min=0) * p + cols)[has]
        for pool in (s["k"], s["v"]):
            flat = pool.view(pool.shape[0], -1, *pool.shape[3:])
            flat[:, b] = flat[:, a]
        return _pages_out(s)
    # compaction: the live pages behind the first `live` places move into the holes before them
    used = refs > 0
    live = used.sum()
    index = torch.arange(refs.numel(), device=refs.device)
    a, b = index[used & (index >= live)], index[~used & (index < live)]
    to = index.clone()
    to[a] = b
    for pool in (s["k"], s["v"]):
        pool[:, b] = pool[:, a]
    refs[b] = refs[a]
    refs[a] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table))
    return _pages_out(s)


def _take(table, refs, slots, have, want, most):
    """The lowest free pages, in the slots' order, for places [have, want) of their rows."""
    need = want - have
    first = need.cumsum(0) - need
    free = torch.sort((refs > 0).to(torch.int8), stable=True).indices  # free ones first, lowest first
    j = torch.arange(most, device=table.device)
    ok = (j < need[:, None]).flatten()
    page = free[(first[:, None] + j).clamp(max=free.numel() - 1)].flatten()
    col = (have[:, None] + j).clamp(max=table.shape[1] - 1).flatten()
    row = slots[:, None].expand(-1, most).flatten()
    row, col, page = row[ok], col[ok], page[ok]
    table[row, col] = page.int()
    refs[page] = 1


def _pages_out(s, **more):
    return dict(k=s["k"], v=s["v"], table=s["table"], lens=s["lens"], refs=s["refs"], grown=s["grown"], **more)


# ------------------------------------------------------------------------- least work
def work(case):
    size = 4 if case.get("dtype") == FP32 else 2
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        if case["mode"] == "serve8":
            groups = case["dim"] // (case["group"] or case["dim"])
            return dict(bytes=n * (size * (3 if case["residual"] else 1) + 1) + 4 * case["rows"] * groups
                        + size * case["dim"], flops=8 * n)
        # forward x (r) -> y (h); backward dy (dh) -> dx, with the stream as one more input
        tensors = 4 + 3 if case["residual"] else 2 + 2
        return dict(bytes=n * size * tensors + 2 * size * case["dim"], flops=20 * n)
    if case["op"] == "rotary":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        ways = 4 if case["mode"] == "train" else 2
        return dict(bytes=n * size * ways + 8 * case["tokens"], flops=3 * n * ways // 2)
    if case["op"] == "attention":
        b, d = case["seqs"], case["head_dim"]
        mid_new = (case["new"] + 1) / 2 if case["ragged_new"] else case["new"]
        mid_kv = (case["kv_min"] + case["kv_max"]) / 2
        new = case["new"] + (b - 1) * mid_new
        kv = case["kv_max"] + (b - 1) * max(mid_kv, mid_new)
        seen = case["new"] * (case["kv_max"] - (case["new"] - 1) / 2) + \
            (b - 1) * mid_new * (max(mid_kv, mid_new) - (mid_new - 1) / 2)
        return dict(bytes=2 * kv * case["kv_heads"] * d * size + 2 * new * case["heads"] * d * size
                    + 4 * new * case["heads"], flops=4 * seen * case["heads"] * d)
    token = case["kv_heads"] * case["head_dim"] * size
    slots = 2 * case["seqs"]
    meta = 4 * (slots * (case["held"] + 2 + -(-case["new"] // case["page"])) + case["pages"])
    if case["mode"] == "append":
        new = case["new"] + (case["seqs"] - 1) * (case["new"] + 1) / 2
        return dict(bytes=2 * 2 * new * token + meta, flops=0)
    stay = case["seqs"] - case["seqs"] // 3
    if case["mode"] == "fork":
        return dict(bytes=2 * 2 * case["layers"] * stay * (case["page"] / 2) * token + meta, flops=0)
    live = min(case["pages"], stay * 0.75 * case["held"])
    moved = live * (1 - live / case["pages"])
    return dict(bytes=2 * 2 * case["layers"] * moved * case["page"] * token + meta, flops=0)


# ------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "rotary": _exact_rotary, "attention": _exact_attention,
                "pages": _exact_pages}[case["op"]](s)


def _exact_norm(s):
    c = s["case"]
    h = (s["x"].double() + s["r"].double()).to(s["x"].dtype) if c["residual"] else s["x"]
    hd, w = h.double(), s["w"].double()
    root = (hd.pow(2).sum(-1, keepdim=True) / c["dim"] + s["eps"]).sqrt()
    y = hd / root * w
    if c["mode"] == "serve8":
        g = c["group"] or c["dim"]
        parts = y.reshape(c["rows"], c["dim"] // g, g)
        scale = parts.abs().max(-1).values / E4M3_MAX
        # the nearest of the 8-bit values: 3 bits behind the leading one, steps of 2^-9 at least
        z = parts / scale[..., None]
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
        y = (torch.round(z / step) * step * scale[..., None]).reshape(c["rows"], c["dim"])
        out = dict(y=y, scale=scale)
        return dict(out, h=h.double()) if c["residual"] else out
    dy = s["dy"].double()
    dn = dy * w
    # d/dh of h / root: 1 / root - h h^T / (dim root^3)
    dx = dn / root - hd * (dn * hd).sum(-1, keepdim=True) / (c["dim"] * root.pow(3))
    dw = (dy * (hd / root)).sum(0)
    if c["residual"]:
        dx = dx + s["dh"].double()
        return dict(y=y, h=h.double(), dx=dx, dr=dx, dw=dw)
    return dict(y=y, dx=dx, dw=dw)


def _exact_rotary(s):
    c, rd = s["case"], s["case"]["rotary_dim"]

    def turned(x, sign):
        # each pair as one complex number, times magnitude * e^(i * angle)
        pair = x[..., :rd].double()
        a, b = (pair[..., 0::2], pair[..., 1::2]) if c["interleaved"] else pair.split(rd // 2, -1)
        angle = sign * s["pos"].double()[:, None, None] * s["inv"]
        z = torch.complex(a, b) * torch.polar(torch.full_like(angle, s["magnitude"]), angle)
        y = torch.stack([z.real, z.imag], -1 if c["interleaved"] else -2).flatten(-2)
        return torch.cat([y, x[..., rd:].double()], -1)

    out = dict(q=turned(s["q"], 1.0), k=turned(s["k"], 1.0))
    if c["mode"] == "train":
        out.update(dq=turned(s["dq"], -1.0), dk=turned(s["dk"], -1.0))
    return out


def _exact_attention(s):
    c, q = s["case"], s["q"]
    t, hq, d = q.shape
    g = hq // c["kv_heads"]
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.zeros(hq, t, dtype=torch.float64, device=q.device)
    for b in range(c["seqs"]):
        n, kv = cu[b + 1] - cu[b], lens[b]
        rows = s["table"][b, :-(-kv // c["page"])].long()
        seen = torch.arange(kv, device=q.device) <= torch.arange(kv - n, kv, device=q.device)[:, None]
        for h in range(c["kv_heads"]):
            k = s["k"][rows, :, h].reshape(-1, d)[:kv].double()
            v = s["v"][rows, :, h].reshape(-1, d)[:kv].double()
            for j in range(h * g, (h + 1) * g):
                a = q[cu[b]:cu[b + 1], j].double() @ k.t() / math.sqrt(d)
                a.masked_fill_(~seen, -math.inf)
                total = torch.logsumexp(a, -1)
                out[cu[b]:cu[b + 1], j] = torch.exp(a - total[:, None]) @ v
                lse[j, cu[b]:cu[b + 1]] = total
    return dict(out=out, lse=lse)


def _exact_pages(s):
    """The same step, page by page on the host. What is returned are copies and whole
    numbers, so the floating values are the inputs' own."""
    c, p = s["case"], s["case"]["page"]
    table, lens, refs, grown = (s[n].cpu().tolist() for n in ("table", "lens", "refs", "grown"))
    more, frm, to = {}, [], []

    def lowest():
        page = refs.index(0)
        refs[page] = 1
        return page

    if c["mode"] == "append":
        cu, positions, cells = s["cu"].tolist(), [], []
        for b, slot in enumerate(s["slots"].tolist()):
            n = cu[b + 1] - cu[b]
            for pos in range(lens[slot], lens[slot] + n):
                if table[slot][pos // p] < 0:
                    table[slot][pos // p] = lowest()
                positions.append(pos)
                cells.append(table[slot][pos // p] * p + pos % p)
            lens[slot] += n
            grown[slot] = n
        cells = torch.tensor(cells, device="cuda")
        for pool, new in ((s["k"], s["new_k"]), (s["v"], s["new_v"])):
            pool[0].view(-1, *pool.shape[3:])[cells] = new
        more["positions"] = _ints(positions)
    else:
        for slot in s["leave"].tolist():
            for j, page in enumerate(table[slot]):
                if page >= 0:
                    refs[page] -= 1
                table[slot][j] = -1
            lens[slot] = grown[slot] = 0
    if c["mode"] == "fork":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            for j in range(lens[a] // p):
                table[b][j] = table[a][j]
                refs[table[a][j]] += 1
            lens[b], grown[b] = lens[a], 0
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            if lens[a] % p:
                j = lens[a] // p
                table[b][j] = lowest()
                frm += [table[a][j] * p + i for i in range(lens[a] % p)]
                to += [table[b][j] * p + i for i in range(lens[a] % p)]
    if c["mode"] == "compact":
        live = sum(r > 0 for r in refs)
        holes = [i for i in range(live) if refs[i] == 0]
        moving = [i for i in range(live, len(refs)) if refs[i] > 0]
        new = dict(zip(moving, holes))
        for i, j in new.items():
            refs[j], refs[i] = refs[i], 0
            frm += range(i * p, i * p + p)
            to += range(j * p, j * p + p)
        table = [[new.get(x, x) for x in row] for row in table]
    if frm:
        frm, to = torch.tensor(frm, device="cuda"), torch.tensor(to, device="cuda")
        for pool in (s["k"], s["v"]):
            flat = pool.view(pool.shape[0], -1, *pool.shape[3:])
            flat[:, to] = flat[:, frm]
    return dict(k=s["k"], v=s["v"], table=_ints(table), lens=_ints(lens), refs=_ints(refs), grown=_ints(grown), **more)
