"""Sampling several answers to a prompt and training on them, as a model's user does it: served
over forked sequences whose prompt is read once, tokens chosen among the alternatives, their log
probabilities taken again by the training model, and the gradient of a loss of these.

The bound is that of test_models_gpu.py: the kernels round no more often than the model's plain
16-bit operators, so their distance from the same model in 64 bits is at most half as much again
as the plain 16-bit model's.
"""
import pytest
import torch
import torch.nn.functional as F

from test_token_logprobs_gpu import close, definition

pytestmark = pytest.mark.gpu

VOCAB, DIM, LAYERS, HEADS, KV, D = 211, 256, 2, 8, 4, 64


def _model(dtype, fused=False, qk_norm=True):
    from multi_gpu_flashattention_b200 import RingTransformerLM
    torch.manual_seed(0)
    m = RingTransformerLM(VOCAB, DIM, LAYERS, HEADS, KV, head_dim=D, mlp_mult=2, fused_ops=fused,
                          qk_norm=qk_norm, fused_loss=fused)
    torch.nn.init.normal_(m.embed.weight, std=0.5)
    for name, p in m.named_parameters():
        if "norm" in name:
            torch.nn.init.normal_(p, 1.0, 0.2)
    return m.to("cuda", dtype)


def _exact(model, ids):
    """Logits of ids [S] from the parameters in 64 bits, with differentiable copies."""
    P = {n: p.detach().double().requires_grad_() for n, p in model.named_parameters()}
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
        q, k = rot(norm(q, W("q_norm"))), rot(norm(k, W("k_norm")))
        k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) / D ** 0.5
        a = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(hide, float("-inf")), -1), v)
        x = x + a.reshape(S, -1) @ W("wo").t()
        h = norm(x, W("norm2"))
        x = x + (F.silu(h @ W("w1").t()) * (h @ W("w3").t())) @ W("w2").t()
    return norm(x, P["norm.weight"]) @ P["embed.weight"].t(), P


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _off(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


def _layout(n):
    from multi_gpu_flashattention_b200 import RingLayout
    return RingLayout("contiguous", n, 1, mask="causal")


def _sample(model, prompt, answers, steps, shared=True):
    """Sequences [answers, prompt + steps], and what serving said of the sampled tokens."""
    from multi_gpu_flashattention_b200 import token_logprobs
    n = prompt.numel()
    cache = model.make_cache(pages=200, page_size=16, slots=answers + 1, max_tokens=n + steps + 16)
    logits = model.serve(prompt, cache, _ints([0]), _ints([0, n]), n)[-1:]
    cache.fork([0] * answers, list(range(1, answers + 1)))
    slots, cu = _ints(list(range(1, answers + 1))), _ints(list(range(answers + 1)))
    groups = _ints([0, answers]) if shared else None
    g = torch.Generator("cuda").manual_seed(3)
    logits = logits.expand(answers, -1)
    seqs, lps, ents, all_logits = [prompt.expand(answers, -1)], [], [], []
    for _ in range(steps):
        r = token_logprobs(logits, torch.zeros(answers, dtype=torch.int64, device="cuda"), top=5)
        pick = torch.multinomial(r.top_logprobs.exp(), 1, generator=g)
        tokens = r.top_indices.gather(1, pick)[:, 0]
        r = token_logprobs(logits, tokens)
        lps.append(r.logprobs)
        ents.append(r.entropy)
        all_logits.append(logits)
        seqs.append(tokens[:, None])
        logits = model.serve(tokens, cache, slots, cu, 1, cu_groups=groups)
    return torch.cat(seqs, 1), torch.stack(lps, 1), torch.stack(ents, 1), torch.stack(all_logits, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sampled_answers_and_the_training_model_agree(dtype):
    from multi_gpu_flashattention_b200 import token_logprobs
    model, plain = _model(dtype, fused=True), _model(dtype)
    prompt = torch.randint(0, VOCAB, (150,), generator=torch.Generator().manual_seed(1)).cuda()
    steps, answers = 9, 12
    seqs, lps, ents, logits = _sample(model, prompt, answers, steps)
    n = prompt.numel()
    for b in (0, 5, 11):
        ids = seqs[b]
        exact, P = _exact(model, ids)
        lay = _layout(ids.numel())
        # serving, against the plain 16-bit model's distance from 64 bits
        far = _off(plain(ids[None], lay)[0, n - 1:-1], exact[n - 1:-1])
        assert _off(logits[b], exact[n - 1:-1]) <= 1.5 * far
        # training: the sampled tokens' log probabilities, the prompt's counting for nothing
        targets = torch.full_like(ids, -100)
        targets[n - 1:-1] = ids[n:]
        r = model.token_logprobs(ids[None], targets[None], lay, top=3)
        want = torch.log_softmax(exact, -1)
        want_lp = want[torch.arange(n - 1, ids.numel() - 1), ids[n:]]
        want_h = -(want.exp() * want).sum(-1)
        assert (r.logprobs[0, :n - 1] == 0).all() and r.logprobs[0, -1] == 0
        # a logprob is off by at most twice the row's largest error of a logit
        worst = 2 * 1.5 * (plain(ids[None], lay)[0].double() - exact).abs().amax(-1)
        # (the chance of the single roundings: as much again)
        assert ((r.logprobs[0, n - 1:-1] - want_lp).abs() <= 2 * worst[n - 1:-1]).all()
        assert ((lps[b] - want_lp).abs() <= 2 * worst[n - 1:-1]).all()
        assert ((r.entropy[0] - want_h).abs() <= 2 * worst * want.abs().amax(-1)).all()
        # The gradient of a loss that weighs the tokens apart, at these logits. (This model's
        # sampled tokens have p = 1 - e^-66: what reaches its parameters are the others' p, which
        # errors of the logits multiply by their exponential, so no multiple of the plain model's
        # distance bounds it; the kernel's own tolerance does.)
        x = model(ids[None], lay)[0].detach().requires_grad_()
        weight = torch.linspace(-1, 1, ids.numel(), device="cuda")
        r = token_logprobs(x, targets)
        dx, = torch.autograd.grad(-(weight * r.logprobs).sum() - 0.01 * r.entropy.sum(), x)
        d = definition(x.detach(), targets, -weight, torch.full_like(weight, -0.01))
        close(dx, d["dx"], d["dx_err"])


def test_gradients_of_a_sampling_loss():
    """Of the parameters, for a loss that weighs the tokens apart and an entropy bonus, where the
    distributions are broad."""
    model, plain = _model(torch.bfloat16, fused=True), _model(torch.bfloat16)
    for m in (model, plain):
        with torch.no_grad():
            m.embed.weight.mul_(0.1)
    ids = torch.randint(0, VOCAB, (160,), generator=torch.Generator().manual_seed(11)).cuda()
    lay = _layout(160)
    targets = torch.cat([ids[1:], ids.new_tensor([-100])])
    targets[:100] = -100
    weight = torch.linspace(-1, 1, 160, device="cuda")

    def loss(logprobs, entropy):
        return -(weight * logprobs).sum() - 0.01 * entropy.sum()

    def of(logits):
        lp = torch.log_softmax(logits, -1)
        picked = torch.where(targets >= 0, lp.gather(1, targets.clamp(min=0)[:, None])[:, 0], torch.zeros_like(lp[:, 0]))
        return loss(picked, -(lp.exp() * lp).sum(-1))

    r = model.token_logprobs(ids[None], targets[None], lay)
    params = dict(model.named_parameters())
    ours = torch.autograd.grad(loss(r.logprobs[0], r.entropy[0]), list(params.values()))
    exact, P = _exact(model, ids)
    exact_g = torch.autograd.grad(of(exact), [P[k] for k in params])
    plain_g = torch.autograd.grad(of(plain(ids[None], lay)[0].float()), list(plain.parameters()))
    flat = lambda gs: torch.cat([x.double().flatten() for x in gs])
    assert _off(flat(ours), flat(exact_g)) <= 1.5 * _off(flat(plain_g), flat(exact_g))


def test_shared_and_apart_serve_alike():
    """With and without cu_groups: the same tokens sampled, logits within the plain model's error."""
    model = _model(torch.bfloat16, fused=True)
    prompt = torch.randint(0, VOCAB, (100,), generator=torch.Generator().manual_seed(2)).cuda()
    a, b = _sample(model, prompt, 20, 1, shared=True), _sample(model, prompt, 20, 1, shared=False)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])  # of the prompt alone
    cache = model.make_cache(100, 16, 8, 300)
    model.serve(prompt, cache, _ints([0]), _ints([0, 100]), 100)
    cache.fork([0] * 7, list(range(1, 8)))
    ids = torch.arange(8, device="cuda") * 11
    cu, slots = _ints(list(range(9))), _ints(list(range(8)))
    free, lens = cache.free_pages(), cache.lens.clone()
    one = model.serve(ids, cache, slots, cu, 1, cu_groups=_ints([0, 8]))
    for s in range(8):
        exact = _exact(model, torch.cat([prompt, ids[s:s + 1]]))[0][-1]
        plain = _model(torch.bfloat16)(torch.cat([prompt, ids[s:s + 1]])[None], _layout(101))[0, -1]
        assert _off(one[s], exact) <= 1.5 * _off(plain, exact) + 1e-3
    # (each sequence has its own copy of the page that the prompt ends in, with room)
    assert cache.free_pages() == free and torch.equal(cache.lens, lens + 1)


def test_loss_and_its_gradient():
    """fused_loss: the loss in float32 as F.cross_entropy has it, the gradient within the plain
    16-bit model's error."""
    model, plain = _model(torch.bfloat16, fused=True), _model(torch.bfloat16)
    ids = torch.randint(0, VOCAB, (128,), generator=torch.Generator().manual_seed(5)).cuda()
    lay = _layout(128)
    targets = torch.cat([ids[1:], ids.new_tensor([-100])])[None]
    loss = model.loss(ids[None], targets, lay)
    with torch.no_grad():
        logits = model(ids[None], lay)
        want = F.cross_entropy(logits.double()[0], targets[0], ignore_index=-100)
    # 127 log probabilities of some 6, each off by a few steps of float32, and their sum
    assert (loss.double() - want).abs() <= 2e-6 * want
    grads = torch.autograd.grad(loss, list(model.parameters()))
    exact, P = _exact(model, ids)
    names = [n for n, _ in model.named_parameters()]
    exact_g = torch.autograd.grad(F.cross_entropy(exact, targets[0], ignore_index=-100), [P[n] for n in names])
    plain_g = torch.autograd.grad(plain.loss(ids[None], targets, lay), list(plain.parameters()))
    flat = lambda gs: torch.cat([x.double().flatten() for x in gs])
    assert _off(flat(grads), flat(exact_g)) <= 1.5 * _off(flat(plain_g), flat(exact_g))


def test_a_captured_sampling_step():
    """reserve, plan, append, shared attention and log probabilities in one graph, against eager steps."""
    from multi_gpu_flashattention_b200 import token_logprobs
    model = _model(torch.bfloat16, fused=True)
    prompt = torch.randint(0, VOCAB, (70,), generator=torch.Generator().manual_seed(7)).cuda()
    slots, cu, groups = _ints([1, 2, 3, 4]), _ints([0, 1, 2, 3, 4]), _ints([0, 4])

    def fresh():
        cache = model.make_cache(60, 16, 5, 120)
        model.serve(prompt, cache, _ints([0]), _ints([0, 70]), 70)
        cache.fork([0] * 4, [1, 2, 3, 4])
        return cache

    def step(cache, ids):
        logits = model.serve(ids, cache, slots, cu, 1, cu_groups=groups)
        return token_logprobs(logits, ids, top=2)

    ids = torch.tensor([3, 5, 7, 9], device="cuda")
    caches = [fresh(), fresh()]
    step(fresh(), ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0], ids)
    for i in range(12):
        ids.copy_(torch.tensor([3, 5, 7, 9], device="cuda") * (i + 1) % VOCAB)
        graph.replay()
        want = step(caches[1], ids)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(caches[0].lens, caches[1].lens)


def test_a_forked_sequence_without_room(monkeypatch):
    """One of a group's sequences gets no page, which is known before the first layer's append:
    the others are served as in a step in which all had room, its logits are NaN."""
    from multi_gpu_flashattention_b200 import KernelStatusError, PagedKVCache
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    model = _model(torch.bfloat16, fused=True)
    prompt = torch.randint(0, VOCAB, (64,), generator=torch.Generator().manual_seed(13)).cuda()
    append, attend = PagedKVCache.append, PagedKVCache.attend

    def late(f):
        def call(self, *a, **kw):  # what reserve() reported has arrived
            torch.cuda.synchronize()
            return f(self, *a, **kw)
        return call

    monkeypatch.setattr(PagedKVCache, "append", late(append))
    monkeypatch.setattr(PagedKVCache, "attend", late(attend))
    ids, got = torch.tensor([1, 2, 3, 4], device="cuda"), {}
    for pages in (8, 7):  # the prompt's 4, and 4 for the sequences' new tokens
        cache = model.make_cache(pages, 16, 4, 96)
        model.serve(prompt, cache, _ints([0]), _ints([0, 64]), 64)
        cache.fork([0] * 3, [1, 2, 3])
        check_errors()
        got[pages] = model.serve(ids, cache, _ints([0, 1, 2, 3]), _ints([0, 1, 2, 3, 4]), 1, cu_groups=_ints([0, 4]))
    assert torch.isnan(got[7][3]).all() and torch.isfinite(got[8]).all()
    with pytest.raises(KernelStatusError, match="too few free pages"):
        check_errors()
    # (the refused one's limits what is shared to the pages before its last token)
    exact = [_exact(model, torch.cat([prompt, ids[i:i + 1]]))[0][-1] for i in range(3)]
    plain = _model(torch.bfloat16)
    for i in range(3):
        far = _off(plain(torch.cat([prompt, ids[i:i + 1]])[None], _layout(65))[0, -1], exact[i])
        assert _off(got[7][i], exact[i]) <= 1.5 * far + 1e-3


def test_training_with_normed_heads_under_autocast():
    """A stream in 32 bits, products in 16, with and without the kernels: gradients of the fused
    model as far from 64 bits as the plain model's."""
    ids = torch.randint(0, VOCAB, (130,), generator=torch.Generator().manual_seed(17)).cuda()
    lay = _layout(129)
    offs = {}
    for fused in (False, True):
        model = _model(torch.float32, fused)
        with torch.autocast("cuda", torch.bfloat16):
            out = model(ids[None, :-1], lay)[0]
        F.cross_entropy(out.float(), ids[1:]).backward()
        logits, P = _exact(model, ids[:-1])
        names = [n for n, _ in model.named_parameters()]
        grads = torch.autograd.grad(F.cross_entropy(logits, ids[1:]), [P[n] for n in names])
        offs[fused] = {n: _off(p.grad, g) for (n, p), g in zip(model.named_parameters(), grads)}
    plain = sum(offs[False].values()) / len(offs[False])
    for n, o in offs[True].items():
        assert o <= 1.5 * max(offs[False][n], plain), (n, o, offs[False][n], plain)


def test_norms_of_queries_and_keys_have_an_eps_of_their_own():
    """Trained on the kernels and served: as far from the formulas as the plain model, for an eps of
    the keys that counts; each eps taken for the other's would be off by more."""
    ids = torch.randint(0, VOCAB, (90,), generator=torch.Generator().manual_seed(19)).cuda()
    plain, fused = _model(torch.bfloat16), _model(torch.bfloat16, fused=True)
    for m in (plain, fused):
        for b in m.blocks:
            b.k_norm.eps = 0.5
    wide = _model(torch.bfloat16).double()
    for b in wide.blocks:
        b.k_norm.eps = 0.5
    want = _with_eps(wide, ids, 1e-6, 0.5)
    far = _off(plain(ids[None], _layout(90))[0], want)
    assert _off(_with_eps(wide, ids, 1e-6, 1e-6), want) > 4 * far and _off(_with_eps(wide, ids, 0.5, 0.5), want) > 4 * far
    assert _off(fused(ids[None], _layout(90))[0], want) <= 1.5 * far
    cache = fused.make_cache(8, 16, 2, 128)
    assert _off(fused.serve(ids, cache, _ints([1]), _ints([0, 90]), 90), want) <= 1.5 * far


def _with_eps(model, ids, q_eps, k_eps):
    """_exact()'s logits with other eps in the heads' norms."""
    import torch as t
    P = {n: p.detach() for n, p in model.named_parameters()}
    norm = lambda x, w, eps=1e-6: x * t.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    S = ids.numel()
    ang = t.arange(S, device="cuda", dtype=t.float64)[:, None] * 10000.0 ** (-t.arange(0, D, 2, device="cuda", dtype=t.float64) / D)
    z = t.polar(t.ones_like(ang), ang)[:, None]
    rot = lambda x: t.view_as_real(t.complex(*x.split(D // 2, -1)) * z).transpose(-1, -2).flatten(-2)
    x = P["embed.weight"][ids]
    hide = t.ones(S, S, dtype=t.bool, device="cuda").triu(1)
    for i in range(LAYERS):
        W = lambda n: P[f"blocks.{i}.{n}.weight"]
        h = norm(x, W("norm1"))
        q, k, v = ((h @ W(n).t()).view(S, -1, D) for n in ("wq", "wk", "wv"))
        q, k = rot(norm(q, W("q_norm"), q_eps)), rot(norm(k, W("k_norm"), k_eps))
        k, v = (y.repeat_interleave(HEADS // KV, 1) for y in (k, v))
        s = t.einsum("qhd,khd->hqk", q, k) / D ** 0.5
        x = x + t.einsum("hqk,khd->qhd", t.softmax(s.masked_fill(hide, float("-inf")), -1), v).reshape(S, -1) @ W("wo").t()
        h = norm(x, W("norm2"))
        x = x + (F.silu(h @ W("w1").t()) * (h @ W("w3").t())) @ W("w2").t()
    return norm(x, P["norm.weight"]) @ P["embed.weight"].t()
