"""Operators of sampling several answers to a prompt and of training on them, measured over
the range in which they are used.

    heads      norms of each query and key head with the rotary positions in the same pass:
               a training step (forward and gradients), or serving
    append     the same (or the positions alone) on the way into a paged cache: queries
               returned, keys and values written to their pages
    shared     attention over a paged cache for sequences that hold the same pages of a long
               prefix, which is read once for all of them
    logprobs   log probabilities of given tokens and the distributions' entropy: a training
               step (forward and gradients), or serving with the top alternatives

`run` computes each in its plain form (elementary torch operations in 32 bits), or,
where `own` is true, calls the package's operators. `exact` gives the same outputs in
64 bits.
"""
import math

import torch

own = False

BF16, FP16, FP32 = "bfloat16", "float16", "float32"
IGNORE = -100
EPS = 1e-6


# ------------------------------------------------------------------------- cases
def listed():
    return [
        # One layer's heads in training: 16384 tokens, 32 query and 8 key heads of 128.
        dict(name="heads train 16384 tokens", op="heads", mode="train", tokens=16384, heads=32,
             kv_heads=8, head_dim=128, rotary_dim=128, interleaved=False, dtype=BF16),
        # Half of a 64-wide head rotated, neighbouring pairs, an odd number of tokens.
        dict(name="heads train 1537 tokens fp16", op="heads", mode="train", tokens=1537, heads=6,
             kv_heads=2, head_dim=64, rotary_dim=32, interleaved=True, dtype=FP16),
        # Serving: eight decoding sequences.
        dict(name="heads serve 8 tokens", op="heads", mode="serve", tokens=8, heads=32,
             kv_heads=8, head_dim=128, rotary_dim=128, interleaved=False, dtype=BF16),
        # A decoding step of 64 sequences: one token each, normed heads.
        dict(name="append 64x1", op="append", seqs=64, new=1, held=200, page=64, heads=32,
             kv_heads=8, head_dim=128, rotary_dim=128, interleaved=False, norm=True, dtype=BF16),
        # Prompts: ragged chunks of 16 sequences, positions alone.
        dict(name="append 16x1024", op="append", seqs=16, new=1024, held=100, page=64, heads=32,
             kv_heads=8, head_dim=128, rotary_dim=128, interleaved=False, norm=False, dtype=BF16),
        # Chunks of odd lengths, heads of 64, short pages.
        dict(name="append 5x333 fp16", op="append", seqs=5, new=333, held=70, page=16, heads=8,
             kv_heads=8, head_dim=64, rotary_dim=48, interleaved=False, norm=True, dtype=FP16),
        # 128 answers to one prompt of 32768 tokens, up to 512 tokens in, a token each.
        dict(name="shared 128 of 32768", op="shared", groups=1, members=128, new=1, ragged_new=False,
             prefix=32768, prefix_min=32768, tail=512, heads=32, kv_heads=8, head_dim=128, page=64,
             dtype=BF16),
        # Eight prompts of 2000 to 8000 tokens with up to eight answers each.
        dict(name="shared 8 groups of 8", op="shared", groups=8, members=8, new=1, ragged_new=False,
             prefix=8000, prefix_min=2000, tail=512, heads=32, kv_heads=8, head_dim=128, page=64,
             dtype=BF16),
        # Three answers to one prompt, a few proposed tokens each, heads of 64.
        dict(name="shared 3 of 1500 fp16", op="shared", groups=1, members=3, new=5, ragged_new=True,
             prefix=1500, prefix_min=1500, tail=90, heads=14, kv_heads=2, head_dim=64, page=16,
             dtype=FP16),
        # A training batch's loss: 4096 tokens over 131072 entries.
        dict(name="logprobs train 4096x131072", op="logprobs", mode="train", rows=4096, vocab=131072,
             top=0, dtype=BF16),
        # An odd number of rows and of entries, in fp32.
        dict(name="logprobs train 1021x50001 fp32", op="logprobs", mode="train", rows=1021,
             vocab=50001, top=0, dtype=FP32),
        # A sampling step of 64 sequences, with the 20 likeliest alternatives.
        dict(name="logprobs serve 64x131072", op="logprobs", mode="serve", rows=64, vocab=131072,
             top=20, dtype=BF16),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["heads", "append", "shared", "shared", "logprobs"])
    kv = rng.choice([1, 2, 4, 8])
    head_dim = rng.choice([64, 128])
    rotary_dim = rng.choice([head_dim, head_dim // 2, 2 * rng.randint(1, head_dim // 2)])
    if op == "heads":
        dtype = rng.choice([BF16, FP16, FP32])
        return dict(op=op, mode=rng.choice(["train", "train", "serve"]), heads=kv * rng.choice([1, 2, 4]),
                    kv_heads=kv, tokens=_log(rng, 1, 8192 if dtype == FP32 else 16384), head_dim=head_dim,
                    rotary_dim=rotary_dim, interleaved=rng.random() < 0.4, dtype=dtype)
    if op == "append":
        seqs = _log(rng, 1, 64)
        return dict(op=op, seqs=seqs, new=rng.choice([1, _log(rng, 2, 8192 // seqs)]),
                    held=_log(rng, 1, 200), page=rng.choice([16, 32, 64, 128]),
                    heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, head_dim=head_dim,
                    rotary_dim=rotary_dim, interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.6, dtype=rng.choice([BF16, FP16]))
    if op == "shared":
        heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
        new = rng.choice([1, 1, 1, _log(rng, 2, 16)])
        groups = _log(rng, 1, 8)
        members = _log(rng, 1, max(1, 128 // (groups * new)))
        # scores of a pass stay below the largest listed case's
        most = min(32768 // groups, 128 * 32 * 32768 // (groups * members * new * heads))
        prefix = _log(rng, 17, most)
        return dict(op=op, groups=groups, members=members, new=new,
                    ragged_new=new > 1 and rng.random() < 0.7, prefix=prefix,
                    prefix_min=rng.randint(1, prefix), tail=_log(rng, new, 512), heads=heads,
                    kv_heads=kv, head_dim=head_dim, page=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice([BF16, FP16]))
    vocab = _log(rng, 100, 131072)
    mode, dtype = rng.choice(["train", "serve"]), rng.choice([BF16, FP16, FP32])
    most = (2048 if dtype == FP32 else 4096) * 131072 // vocab
    return dict(op=op, mode=mode, vocab=vocab, rows=_log(rng, 1, min(16384, most) if mode == "train" else 256),
                top=rng.randint(0, 20) if mode == "serve" else 0, dtype=dtype)


# ------------------------------------------------------------------------- inputs
def _dtype(case):
    return getattr(torch, case["dtype"])


def _rng(seed):
    """A generator on the host (sizes, places) and one on the device (values)."""
    return torch.Generator().manual_seed(seed), torch.Generator("cuda").manual_seed(seed)


def _randn(shape, dtype, gen, std=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(0.0, std, generator=gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inv_freq(rotary_dim):
    """Radians a position of each rotated pair, in 64 bits."""
    return (10000.0 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)).cuda()


def _ragged(most, n, shape_seed):
    """1 to `most`, n times, the first `most`: the same for every seed, since they give the
    outputs' shapes."""
    host = torch.Generator().manual_seed(shape_seed)
    return [most] + torch.randint(1, most + 1, (n - 1,), generator=host).tolist()


def _sums(values):
    out = [0]
    for a in values:
        out.append(out[-1] + a)
    return out


def prepare(case, seed):
    return {"heads": _prepare_heads, "append": _prepare_append, "shared": _prepare_shared,
            "logprobs": _prepare_logprobs}[case["op"]](case, seed)


def _weights(case, gen):
    """The norms' weights, of the inputs' type."""
    return [(1 + 0.1 * torch.randn(case["head_dim"], device="cuda", generator=gen)).to(_dtype(case))
            for _ in range(2)]


def _prepare_heads(case, seed):
    host, gen = _rng(seed)
    dt, t, d = _dtype(case), case["tokens"], case["head_dim"]
    train = case["mode"] == "train"
    s = dict(case=case, inv=_inv_freq(case["rotary_dim"]))
    wq, wk = _weights(case, gen)
    if train:
        s["pos"] = torch.arange(t, dtype=torch.int32, device="cuda")
        s["q"] = _randn((t, case["heads"], d), dt, gen, 1.5).requires_grad_()
        s["k"] = _randn((t, case["kv_heads"], d), dt, gen, 1.5).requires_grad_()
        s["dq"], s["dk"] = _randn(s["q"].shape, dt, gen), _randn(s["k"].shape, dt, gen)
        wq.requires_grad_(), wk.requires_grad_()
    else:
        s["pos"] = torch.randint(0, 131072, (t,), generator=host, dtype=torch.int32).cuda()
        # the columns of one projection
        qkv = _randn((t, case["heads"] + 2 * case["kv_heads"], d), dt, gen, 1.5)
        s["q"], s["k"], _ = qkv.split([case["heads"], case["kv_heads"], case["kv_heads"]], 1)
    s.update(wq=wq, wk=wk)
    return s


def _prepare_append(case, seed):
    """A step behind reserve(): the sequences' lengths count the new tokens, which have their
    pages. The pool's pages lie in any order."""
    host, gen = _rng(seed)
    dt, n, p, d = _dtype(case), case["seqs"], case["page"], case["head_dim"]
    new = _ragged(case["new"], n, n)
    held = torch.randint(0, case["held"] + 1, (n,), generator=host).tolist()
    lens = [a + b for a, b in zip(held, new)]
    width = -(-(case["held"] + case["new"]) // p)
    pages = sum(-(-(case["held"] + a) // p) for a in new)  # for any seed's lengths
    order = torch.randperm(pages, generator=host).tolist()
    slots = torch.randperm(2 * n, generator=host).tolist()[:n]
    table, refs, at = [[-1] * width for _ in range(2 * n)], [0] * pages, 0
    length, grown = [0] * (2 * n), [0] * (2 * n)
    for b, slot in enumerate(slots):
        need = -(-lens[b] // p)
        table[slot][:need] = order[at:at + need]
        at += need
        length[slot], grown[slot] = lens[b], new[b]
    for page in order[:at]:
        refs[page] = 1
    cu = _sums(new)
    qkv = _randn((cu[-1], case["heads"] + 2 * case["kv_heads"], d), dt, gen, 1.5)
    q, k, v = qkv.split([case["heads"], case["kv_heads"], case["kv_heads"]], 1)
    shape = (1, pages, p, case["kv_heads"], d)
    wq, wk = _weights(case, gen)
    pos = [held[b] + i for b in range(n) for i in range(new[b])]
    s = dict(case=case, q=q, k=k, v=v, pos=_ints(pos), slots=_ints(slots), cu=_ints(cu),
             table=_ints(table), lens=_ints(length), refs=_ints(refs), grown=_ints(grown),
             k_pool=_randn(shape, dt, gen), v_pool=_randn(shape, dt, gen),
             inv=_inv_freq(case["rotary_dim"]))
    if case["norm"]:
        s.update(wq=wq, wk=wk)
    return s


def _prepare_shared(case, seed):
    """Sequences forked from their group's prompt: its full pages are held by all, the tokens
    of its last page and their own by each."""
    host, gen = _rng(seed)
    dt, p, d = _dtype(case), case["page"], case["head_dim"]
    sizes = _ragged(case["members"], case["groups"], 7)
    n = sum(sizes)
    new = _ragged(case["new"], n, n) if case["ragged_new"] else [case["new"]] * n
    prefix = torch.randint(case["prefix_min"], case["prefix"] + 1, (case["groups"],), generator=host).tolist()
    prefix[0] = case["prefix"]
    tails = torch.randint(1, case["tail"] + 1, (n,), generator=host).tolist()
    kv, need, full = [], [], []
    for g, size in enumerate(sizes):
        for _ in range(size):
            b = len(kv)
            kv.append(prefix[g] + max(tails[b], new[b]))
            full.append(prefix[g] // p)
            need.append(-(-kv[b] // p) - full[b])
    pool = sum(a // p for a in prefix) + sum(need)
    order = torch.randperm(pool, generator=host).tolist()
    width = -(-(case["prefix"] + case["tail"]) // p)
    table, at, b = [], 0, 0
    for g, size in enumerate(sizes):
        common = order[at:at + prefix[g] // p]
        at += len(common)
        for _ in range(size):
            row = common + order[at:at + need[b]]
            at += need[b]
            b += 1
            table.append(row + [-1] * (width - len(row)))
    cu, cg = _sums(new), _sums(sizes)
    for g, size in enumerate(sizes):
        if size == 1:  # all that a sequence alone held before is its group's
            full[cg[g]] = (kv[cg[g]] - new[cg[g]]) // p
    shape = (pool, p, case["kv_heads"], d)
    return dict(case=case, q=_randn((cu[-1], case["heads"], d), dt, gen), k=_randn(shape, dt, gen),
                v=_randn(shape, dt, gen), table=_ints(table), lens=_ints(kv), cu=_ints(cu),
                groups=_ints(cg), max_new=max(new), max_prefix=max(full) * p,
                max_own=max(a - f * p for a, f in zip(kv, full)),
                max_rows=max(cu[b] - cu[a] for a, b in zip(cg, cg[1:])))


def _prepare_logprobs(case, seed):
    host, gen = _rng(seed)
    dt, n, v = _dtype(case), case["rows"], case["vocab"]
    targets = torch.randint(0, v, (n,), generator=host)
    train = case["mode"] == "train"
    s = dict(case=case, x=_randn((n, v), dt, gen, 2.5).requires_grad_(train))
    if train:  # padding and prompt tokens count for nothing; advantages, and an entropy bonus
        targets[torch.rand(n, generator=host) < 0.1] = IGNORE
        s["dl"] = torch.randn(n, device="cuda", generator=gen)
        s["dh"] = torch.full((n,), 0.01, device="cuda")
    s["t"] = targets.cuda()
    return s


# ------------------------------------------------------------------------- one pass
def run(s):
    return {"heads": _run_heads, "append": _run_append, "shared": _run_shared,
            "logprobs": _run_logprobs}[s["case"]["op"]](s)


def _angles(s):
    angle = s["pos"].double()[:, None] * s["inv"]  # far positions: 64 bits
    return angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]


def _turn(x, cos, sin, c):
    """x's first rotary_dim columns rotated, in 32 bits."""
    rd = c["rotary_dim"]
    xr = x[..., :rd]
    if c["interleaved"]:
        a, b = xr[..., 0::2], xr[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = xr[..., :rd // 2], xr[..., rd // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., rd:]], -1)


def _head_norm(x):
    """x over its heads' root mean squares, and 1 over these, in 32 bits."""
    xf = x.float()
    rstd = torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS)
    return xf * rstd, rstd


def _run_heads(s):
    c = s["case"]
    train = c["mode"] == "train"
    if own:
        from multi_gpu_flashattention_b200 import apply_norm_rotary
        q, k = apply_norm_rotary(s["q"], s["k"], s["pos"], s["inv"], s["wq"], s["wk"], eps=EPS,
                                 interleaved=c["interleaved"])
        if not train:
            return dict(q=q, k=k)
        dq, dk, dwq, dwk = torch.autograd.grad([q, k], [s["q"], s["k"], s["wq"], s["wk"]],
                                               [s["dq"], s["dk"]])
        return dict(q=q, k=k, dq=dq, dk=dk, dwq=dwq, dwk=dwk)
    with torch.no_grad():
        cos, sin = _angles(s)
        out = {}
        for name in ("q", "k"):
            x, w = s[name], s["w" + name].float()
            n, rstd = _head_norm(x)
            out[name] = _turn(n * w, cos, sin, c).to(x.dtype)
            if train:  # the transpose of a rotation is the rotation back
                g = _turn(s["d" + name].float(), cos, -sin, c)
                out["dw" + name] = (g * n).sum((0, 1)).to(x.dtype)
                g = g * w
                out["d" + name] = (rstd * (g - n * (g * n).mean(-1, keepdim=True))).to(x.dtype)
        return out


def _run_append(s):
    c = s["case"]
    if own:
        cache = s.get("cache")
        if cache is None:
            from multi_gpu_flashattention_b200 import PagedKVCache
            cache = s["cache"] = PagedKVCache(s["k_pool"], s["v_pool"], s["table"], s["lens"],
                                              s["refs"], s["grown"])
        q = cache.append(0, s["q"], s["k"], s["v"], s["pos"], s["inv"], s["slots"], s["cu"],
                         q_weight=s.get("wq"), k_weight=s.get("wk"), eps=EPS,
                         interleaved=c["interleaved"])
        return dict(q=q, k=s["k_pool"], v=s["v_pool"])
    cos, sin = _angles(s)
    q, k = s["q"].float(), s["k"].float()
    if c["norm"]:
        q, k = _head_norm(q)[0] * s["wq"].float(), _head_norm(k)[0] * s["wk"].float()
    q, k = _turn(q, cos, sin, c).to(s["q"].dtype), _turn(k, cos, sin, c).to(s["k"].dtype)
    slots, cu, p = s["slots"].long(), s["cu"].long(), c["page"]
    at = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu, at, right=True) - 1
    place = s["lens"][slots][seq].long() - s["grown"][slots][seq] + at - cu[seq]
    cell = s["table"][slots[seq], place // p].long() * p + place % p
    s["k_pool"].view(-1, *k.shape[1:]).index_copy_(0, cell, k)
    s["v_pool"].view(-1, *k.shape[1:]).index_copy_(0, cell, s["v"])
    return dict(q=q, k=s["k_pool"], v=s["v_pool"])


def _run_shared(s):
    c = s["case"]
    if own:
        from multi_gpu_flashattention_b200 import paged_attention, shared_prefix
        plan = shared_prefix(s["table"], s["lens"], s["cu"], s["groups"], c["page"])
        out, lse = paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"],
                                   s["max_new"], shared=plan, return_lse=True)
        return dict(out=out, lse=lse)
    q, m, p, r = s["q"], s["max_new"], c["page"], s["max_rows"]
    t, hq, d = q.shape
    hkv, dev = c["kv_heads"], q.device
    h = hq // hkv
    table, lens, cu, cg = s["table"].long(), s["lens"].long(), s["cu"].long(), s["groups"].long()
    b, g = lens.numel(), cg.numel() - 1
    n_new = cu[1:] - cu[:-1]
    # how many tokens each group's sequences share
    group = torch.searchsorted(cg, torch.arange(b, device=dev), right=True) - 1
    lead = table[cg[:-1]]
    pages = ((table == lead[group]) & (table >= 0)).long().cumprod(-1).sum(-1)
    pages = torch.minimum(pages, (lens - n_new) // p)
    common = torch.full((g,), table.shape[1], device=dev).scatter_reduce(0, group, pages, "amin") * p

    def attend(rows, hidden, k, v):
        """Of `rows` [batch, tokens] of q over keys [batch, keys, hkv, d]: the scores' largest
        and, relative to it, the sums of exponentials and of these times the values."""
        n = rows.shape[1]
        x = q[rows].float().view(-1, n, hkv, h, d).permute(0, 2, 1, 3, 4).reshape(-1, hkv, n * h, d)
        a = (x @ k.float().permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(d)).view(-1, hkv, n, h, k.shape[1])
        a.masked_fill_(hidden[:, None, :, None, :], float("-inf"))
        top = a.amax(-1, keepdim=True).clamp(min=-1e30)
        e = a.sub_(top).exp_()
        o = (e.view(-1, hkv, n * h, k.shape[1]) @ v.float().permute(0, 2, 1, 3)).view(-1, hkv, n, h, d)
        return [y.permute(0, 2, 1, 3, 4).reshape(-1, n, hq, y.shape[-1])
                for y in (top, e.sum(-1, keepdim=True), o)]

    at = torch.arange(t, device=dev)
    seq = torch.searchsorted(cu, at, right=True) - 1
    # a sequence's own keys, behind the shared ones; a token sees itself and all before
    place = common[group][:, None] + torch.arange(s["max_own"], device=dev)
    cell = table.gather(1, (place // p).clamp(max=table.shape[1] - 1)).clamp(min=0) * p + place % p
    i = torch.arange(m, device=dev)
    hidden = place[:, None, :] > (lens - n_new)[:, None, None] + i[:, None]
    k, v = s["k"].view(-1, hkv, d), s["v"].view(-1, hkv, d)
    parts = [y[seq, at - cu[seq]] for y in
             attend((cu[:-1, None] + i).clamp(max=t - 1), hidden, k[cell], v[cell])]
    if s["max_prefix"]:
        place = torch.arange(s["max_prefix"], device=dev)
        cell = lead[:, place // p].clamp(min=0) * p + place % p
        hidden = (place >= common[:, None])[:, None, :].expand(-1, r, -1)
        i = torch.arange(r, device=dev)
        over = attend((cu[cg[:-1], None] + i).clamp(max=t - 1), hidden, k[cell], v[cell])
        over = [y[group[seq], at - cu[cg[group[seq]]]] for y in over]
        top = torch.maximum(parts[0], over[0])
        wa, wb = (parts[0] - top).exp(), (over[0] - top).exp()
        parts = [top, parts[1] * wa + over[1] * wb, parts[2] * wa + over[2] * wb]
    top, total, o = parts
    return dict(out=(o / total).to(q.dtype), lse=(top + total.log()).squeeze(-1).t().contiguous())


def _run_logprobs(s):
    c = s["case"]
    if own:
        from multi_gpu_flashattention_b200 import token_logprobs
        r = token_logprobs(s["x"], s["t"], top=c["top"], ignore_index=IGNORE)
        out = dict(logprobs=r.logprobs, entropy=r.entropy)
        if c["top"]:
            out.update(top_logprobs=r.top_logprobs, top_indices=r.top_indices)
        if c["mode"] == "train":
            out["dx"], = torch.autograd.grad([r.logprobs, r.entropy], [s["x"]], [s["dl"], s["dh"]])
        return out
    with torch.no_grad():
        x, t = s["x"].float(), s["t"]
        top = x.amax(-1, keepdim=True)
        z = x - top
        e = z.exp()
        total = e.sum(-1, keepdim=True)
        log_total = total.log()
        known = t != IGNORE
        at = t.clamp(min=0)[:, None]
        lp = torch.where(known, (z.gather(1, at) - log_total).squeeze(1), torch.zeros_like(top[:, 0]))
        entropy = log_total - (e * z).sum(-1, keepdim=True) / total
        out = dict(logprobs=lp, entropy=entropy.squeeze(1))
        if c["top"]:  # the likeliest first, of equal ones the lowest index
            value, index = torch.sort(x, dim=-1, descending=True, stable=True)
            out.update(top_logprobs=value[:, :c["top"]] - top - log_total, top_indices=index[:, :c["top"]])
        if c["mode"] == "train":
            prob = e / total
            dl = torch.where(known, s["dl"], torch.zeros_like(s["dl"]))[:, None]
            dx = -prob * (dl + s["dh"][:, None] * (z - log_total + entropy))
            dx.scatter_add_(1, at, dl)
            out["dx"] = dx.to(s["x"].dtype)
        return out


# ------------------------------------------------------------------------- least work
def work(case):
    size = 4 if case["dtype"] == FP32 else 2
    if case["op"] == "heads":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        train = case["mode"] == "train"  # x -> y; x, dy -> dx: x is one input
        return dict(bytes=n * size * (4 if train else 2) + 4 * case["tokens"], flops=n * (24 if train else 8))
    if case["op"] == "append":
        new = case["new"] + (case["seqs"] - 1) * (case["new"] + 1) / 2
        d = case["head_dim"]
        return dict(bytes=new * size * d * 2 * (case["heads"] + 2 * case["kv_heads"]) + 4 * new,
                    flops=new * d * (case["heads"] + case["kv_heads"]) * (8 if case["norm"] else 3))
    if case["op"] == "shared":
        d = case["head_dim"]
        n = case["members"] + (case["groups"] - 1) * (case["members"] + 1) / 2
        new = (case["new"] + 1) / 2 if case["ragged_new"] else case["new"]
        prefix = (case["prefix"] + (case["groups"] - 1) * (case["prefix"] + case["prefix_min"]) / 2) / case["groups"]
        tail = max(new, (1 + case["tail"]) / 2)
        token = case["kv_heads"] * d * size
        return dict(bytes=2 * (case["groups"] * prefix + n * tail) * token
                    + n * new * case["heads"] * (2 * d * size + 4),
                    flops=4 * n * new * case["heads"] * d * (prefix + tail - (new - 1) / 2))
    n = case["rows"] * case["vocab"]
    if case["mode"] == "train":
        return dict(bytes=2 * n * size + 24 * case["rows"], flops=16 * n)
    return dict(bytes=n * size + case["rows"] * (16 + 12 * case["top"]), flops=8 * n)


# ------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"heads": _exact_heads, "append": _exact_append, "shared": _exact_shared,
            "logprobs": _exact_logprobs}[case["op"]](s)


def _turned(x, s):
    """Each pair as one complex number, times e^(i * angle)."""
    c, rd = s["case"], s["case"]["rotary_dim"]
    pair = x[..., :rd]
    a, b = (pair[..., 0::2], pair[..., 1::2]) if c["interleaved"] else pair.split(rd // 2, -1)
    angle = s["pos"].double()[:, None, None] * s["inv"]
    z = torch.complex(a, b) * torch.polar(torch.ones_like(angle), angle)
    y = torch.stack([z.real, z.imag], -1 if c["interleaved"] else -2).flatten(-2)
    return torch.cat([y, x[..., rd:]], -1)


def _exact_heads(s):
    out = {}
    for name in ("q", "k"):
        x, w = (s[n].detach().double().requires_grad_() for n in (name, "w" + name))
        y = _turned(x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w, s)
        out[name] = y.detach()
        if s["case"]["mode"] == "train":
            out["d" + name], out["dw" + name] = torch.autograd.grad(y, [x, w], s["d" + name].double())
    return out


def _exact_append(s):
    c, p = s["case"], s["case"]["page"]
    turned = []
    for name in ("q", "k"):
        x = s[name].double()
        if c["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * s["w" + name].double()
        turned.append(_turned(x, s))
    k, v = s["k_pool"].double(), s["v_pool"].double()
    cu, table, pos = s["cu"].tolist(), s["table"].tolist(), s["pos"].tolist()
    cells = [table[slot][pos[i] // p] * p + pos[i] % p
             for b, slot in enumerate(s["slots"].tolist()) for i in range(cu[b], cu[b + 1])]
    cells = torch.tensor(cells, device="cuda")
    k.view(-1, *k.shape[3:])[cells] = turned[1]
    v.view(-1, *v.shape[3:])[cells] = s["v"].double()
    return dict(q=turned[0], k=k, v=v)


def _exact_shared(s):
    """Each sequence by itself over all its keys."""
    c, q = s["case"], s["q"]
    t, hq, d = q.shape
    h = hq // c["kv_heads"]
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.zeros(hq, t, dtype=torch.float64, device=q.device)
    for b, kv in enumerate(lens):
        n = cu[b + 1] - cu[b]
        rows = s["table"][b, :-(-kv // c["page"])].long()
        k = s["k"][rows].flatten(0, 1)[:kv].double().repeat_interleave(h, 1)
        v = s["v"][rows].flatten(0, 1)[:kv].double().repeat_interleave(h, 1)
        a = torch.einsum("ihd,jhd->hij", q[cu[b]:cu[b + 1]].double(), k) / math.sqrt(d)
        a.masked_fill_(torch.arange(kv, device=q.device) > torch.arange(kv - n, kv, device=q.device)[:, None], -math.inf)
        total = torch.logsumexp(a, -1)
        out[cu[b]:cu[b + 1]] = torch.einsum("hij,jhd->ihd", torch.exp(a - total[..., None]), v)
        lse[:, cu[b]:cu[b + 1]] = total
    return dict(out=out, lse=lse)


def _exact_logprobs(s):
    c, out = s["case"], {}
    rows = max(1, (1 << 26) // c["vocab"])  # of a piece
    for i in range(0, c["rows"], rows):
        x = s["x"][i:i + rows].detach().double().requires_grad_()
        t = s["t"][i:i + rows]
        logp = torch.log_softmax(x, -1)
        entropy = -(logp.exp() * logp).sum(-1)
        lp = logp[torch.arange(t.numel(), device=t.device), t.clamp(min=0)] * (t != IGNORE)
        piece = dict(logprobs=lp.detach(), entropy=entropy.detach())
        if c["top"]:
            index = torch.argsort(-x.detach(), dim=-1, stable=True)[:, :c["top"]]
            piece.update(top_logprobs=logp.detach().gather(1, index), top_indices=index)
        if c["mode"] == "train":
            piece["dx"], = torch.autograd.grad([lp, entropy], [x], [s["dl"][i:i + rows].double(),
                                                                    s["dh"][i:i + rows].double()])
        for name, value in piece.items():
            out.setdefault(name, []).append(value)
    return {name: torch.cat(values) for name, values in out.items()}
