"""token_logprobs and its gradient against the definition in 64 bits, and against differences.

Tolerances, fixed before the first run, in steps of float32, u = 2^-24; z = x - max x, and E
is the mean under p. An exponential is off by 2.5 |z| steps (the difference, its product with
log2 e and that constant) and 4 (the 2^x instruction); a sum S of them by the p-weighted
mean of that, by its chain (a thread adds 32 pairs of each of its at most V / 2048 segments;
then joins of lanes, warps and CTAs, 5 + 3 + 3 of them at 6 steps): s = 2.5 E|z| + 4 +
V / 64 + 100 steps. So
  ln S      s + 2 |ln S|
  logprob   that + 2 |z_t| + |ln S| + |logprob|
  entropy   ln S's, and of E|z|, whose terms are |z| times as large:
            2.5 E z^2 + (s + 8) E|z|, and |H| for the difference
  dx        p is off by |z| + 8 + s steps of itself (the exponent's product is exact there),
            A = dl + dh (ln p + H) by 2 |A| + |dh| (ln p's and H's own errors + 2 |ln p|);
            and u of the type, 2^-25 for fp16's subnormals, 1e-37 (1 + |A|) for exponentials
            below 2^-126, which are 0.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def definition(x, t, dl=None, dh=None, ignore=-100):
    """x [N, V], t [N]: logprobs, entropy, dx in 64 bits, and their errors' bounds."""
    xd = x.double()
    V = x.shape[1]
    m = xd.amax(-1, keepdim=True)
    z = xd - m
    e = z.exp()
    S = e.sum(-1, keepdim=True)
    p, ln_s = e / S, S.log()
    finite = z.clamp(min=-1e4)
    ez = (p * finite.abs()).sum(-1, keepdim=True)
    ez2 = (p * finite.square()).sum(-1, keepdim=True)
    lnp = finite - ln_s
    H = -(p * lnp).sum(-1, keepdim=True)
    s = 2.5 * ez + 4 + V / 64 + 100
    ln_err = s + 2 * ln_s.abs()
    h_err = ln_err + 2.5 * ez2 + (s + 8) * ez + H.abs()
    at = t.clamp(0, V - 1).long()[:, None]
    zt = z.gather(1, at)
    lp = zt - ln_s
    lp_err = ln_err + 2 * zt.abs().clamp(max=1e38) + ln_s.abs() + lp.abs().clamp(max=1e38)
    keep = (t != ignore)[:, None]
    out = dict(logprobs=torch.where(keep, lp, torch.zeros_like(lp))[:, 0], entropy=H[:, 0],
               logprobs_err=U * lp_err[:, 0], entropy_err=U * h_err[:, 0],
               lnp=z - ln_s, lnp_err=U * (ln_err + 2 * finite.abs() + ln_s.abs() + lnp.abs()))
    if dl is not None:
        a = torch.where(keep, dl.double()[:, None], torch.zeros_like(lp))
        b = dh.double()[:, None]
        A = a + b * (lnp + H)
        dx = -p * A
        dx.scatter_add_(1, at, a)
        a_err = 2 * A.abs() + b.abs() * (ln_err + h_err + 2 * lnp.abs())
        err = U * p * (A.abs() * (finite.abs() + 8 + s) + a_err)
        err.scatter_add_(1, at, U * 2 * a.abs())
        u = torch.finfo(x.dtype).eps / 2
        out.update(dx=dx, dx_err=err + u * dx.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 0) + 1e-37 * (1 + A.abs()))
    return out


def close(got, ref, err):
    bad = (got.double() - ref).abs() > err
    assert not bad.any(), ((got.double() - ref).abs() - err).max().item()


def top_of(x, k):
    value, index = torch.sort(x.double(), dim=-1, descending=True, stable=True)
    return value[:, :k], index[:, :k]


def check(x, t, top=0, grads=True, seed=0, **kw):
    from multi_gpu_flashattention_b200 import token_logprobs
    g = torch.Generator("cuda").manual_seed(seed)
    dl, dh = torch.randn(x.shape[0], device="cuda", generator=g), torch.randn(x.shape[0], device="cuda", generator=g)
    leaf = x.detach().requires_grad_(grads)
    r = token_logprobs(leaf, t, top=top, **kw)
    d = definition(x, t, dl, dh, **{"ignore": kw.get("ignore_index", -100)})
    assert r.logprobs.dtype == r.entropy.dtype == torch.float32 and r.logprobs.shape == t.shape
    close(r.logprobs, d["logprobs"], d["logprobs_err"])
    close(r.entropy, d["entropy"], d["entropy_err"])
    if top:
        value, index = top_of(x, top)
        assert torch.equal(r.top_indices, index)
        close(r.top_logprobs, d["lnp"].gather(1, index), d["lnp_err"].gather(1, index))
    else:
        assert r.top_logprobs is None and r.top_indices is None
    if grads:
        dx, = torch.autograd.grad([r.logprobs, r.entropy], [leaf], [dl, dh])
        assert dx.dtype == x.dtype and dx.shape == x.shape
        close(dx, d["dx"], d["dx_err"])
    return r


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,V", [(1, 1), (3, 2), (5, 7), (9, 100), (2, 1024), (7, 2040), (6, 2055), (300, 513),
                                 (4, 16384), (3, 16391), (2, 50001), (33, 9999), (1, 131072), (5, 140001)])
def test_against_the_definition(N, V, dtype):
    g = torch.Generator("cuda").manual_seed(V)
    x = (torch.randn(N, V, device="cuda", generator=g) * 3).to(dtype)
    t = torch.randint(0, V, (N,), device="cuda", generator=g)
    if N > 1:
        t[N // 2] = -100
    check(x, t, top=0)
    check(x, t.int(), top=min(V, 1 + V % 32))
    check(x, t, top=min(V, 32), grads=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_any_stride_and_start(dtype):
    """A slice of a padded vocab, rows apart, a start off a 16-byte boundary, columns apart,
    repeated rows, three dimensions; expanded gradients."""
    from multi_gpu_flashattention_b200 import token_logprobs
    base = torch.randn(12, 5000, device="cuda").to(dtype)
    t = torch.randint(0, 4000, (12,), device="cuda")
    for x in (base[:, :4000], base[:, 8:4011], base[:, 3:4300], base[::2, 1:4200], base[:1].expand(12, 5000),
              base.t().contiguous().t()):
        check(x, t[:x.shape[0]], top=5)
    x3 = base[:, :4003].reshape(3, 4, 4003).clone().requires_grad_()
    r = token_logprobs(x3, t.view(3, 4))
    assert r.logprobs.shape == r.entropy.shape == (3, 4)
    dx, = torch.autograd.grad(r.logprobs.sum() - 0.5 * r.entropy.sum(), x3)
    one = torch.ones(12, device="cuda")
    d = definition(x3.detach().view(12, 4003), t, one, -0.5 * one)
    close(dx.view(12, 4003), d["dx"], d["dx_err"])
    row = base[0].clone().requires_grad_()
    r = token_logprobs(row, t[0], top=3)
    assert r.logprobs.shape == () and r.top_indices.shape == (3,)
    r.logprobs.backward()
    d = definition(row.detach()[None], t[:1], one[:1], 0 * one[:1])
    close(row.grad[None], d["dx"], d["dx_err"])


def test_gradient_of_one_output():
    from multi_gpu_flashattention_b200 import token_logprobs
    x = torch.randn(6, 3001, device="cuda").requires_grad_()
    t = torch.randint(0, 3001, (6,), device="cuda")
    one, zero = torch.ones(6, device="cuda"), torch.zeros(6, device="cuda")
    for name, dl, dh in (("logprobs", one, zero), ("entropy", zero, one)):
        r = token_logprobs(x, t, top=2)
        dx, = torch.autograd.grad([getattr(r, name)], [x], [one])
        d = definition(x.detach(), t, dl, dh)
        close(dx, d["dx"], d["dx_err"])
        assert not r.top_logprobs.requires_grad and not r.top_indices.requires_grad


def test_gradient_against_differences():
    """(L(x + hv) - L(x - hv)) / 2h of the kernel's outputs differs from the definition's by the
    outputs' errors over h, and that from the definition's gradient by what 64 bits show."""
    from multi_gpu_flashattention_b200 import token_logprobs
    h = 2.0 ** -5
    x, v = torch.randn(4, 777, device="cuda") * 2, torch.randn(4, 777, device="cuda")
    t = torch.randint(0, 777, (4,), device="cuda")
    dl, dh = torch.randn(4, device="cuda"), torch.randn(4, device="cuda")
    leaf = x.clone().requires_grad_()
    r = token_logprobs(leaf, t)
    dx, = torch.autograd.grad([r.logprobs, r.entropy], [leaf], [dl, dh])
    ours, exact, noise = [], [], 0.0
    for s in (1, -1):
        at = x + s * h * v
        r, d = token_logprobs(at, t), definition(at, t)
        ours.append((dl.double() * r.logprobs + dh.double() * r.entropy).sum())
        exact.append((dl.double() * d["logprobs"] + dh.double() * d["entropy"]).sum())
        noise += (dl.abs() * d["logprobs_err"] + dh.abs() * d["entropy_err"]).sum()
    d = definition(x, t, dl, dh)
    along = (d["dx"] * v).sum()
    # the ends as the kernel sees them are rounded to float32, exactly those that `exact` uses,
    # but are x +- hv only up to a step of them
    ends = (d["dx"].abs() * U * (x.abs() + h * v.abs())).sum() / h
    slope = ((exact[0] - exact[1]) / (2 * h) - along).abs() + noise / (2 * h) + (d["dx_err"] * v.abs()).sum() + ends
    assert ((dx.double() * v).sum() - (ours[0] - ours[1]) / (2 * h)).abs() <= slope


def test_masked_and_extreme_logits():
    """-inf and the type's lowest value as masks, a row with nothing left, one token left, +inf
    and NaN, which stay their row's."""
    from multi_gpu_flashattention_b200 import token_logprobs
    for dtype, V in ((torch.float32, 5000), (torch.bfloat16, 300), (torch.float16, 20000)):
        low, inf = torch.finfo(dtype).min, float("inf")
        x = (torch.randn(10, V, device="cuda") * 2).to(dtype)
        t = torch.randint(100, V, (10,), device="cuda")
        x[0, ::2] = -inf
        x[0, t[0]] = 1.0
        x[1, 50:] = -inf  # the target among them
        x[2, 1:] = -inf
        t[2] = 0
        x[3] = -inf
        x[4, : V // 2] = low
        x[5] = low
        x[6] = torch.finfo(dtype).max
        x[7, 10], x[7, 11] = torch.finfo(dtype).max, low
        x[8, 7] = inf
        x[9, 7] = float("nan")
        leaf = x.clone().requires_grad_()
        r = token_logprobs(leaf, t, top=4)
        dl = torch.ones(10, device="cuda")
        dx, = torch.autograd.grad([r.logprobs, r.entropy], [leaf], [dl, dl])
        ok = [0, 2, 4, 5, 6, 7]
        d = definition(x[ok], t[ok], dl[ok], dl[ok])
        close(r.logprobs[ok], d["logprobs"], d["logprobs_err"])
        close(r.entropy[ok], d["entropy"], d["entropy_err"])
        close(dx[ok], d["dx"], d["dx_err"])
        assert r.logprobs[1] == -inf and torch.isfinite(r.entropy[1]) and torch.isfinite(dx[1]).all()
        assert r.logprobs[3] == -inf and r.entropy[3] == 0 and (dx[3] == 0).all()
        assert r.top_indices[3].tolist() == [0, 1, 2, 3] and (r.top_logprobs[3] == -inf).all()
        assert r.top_indices[5].tolist() == r.top_indices[6].tolist() == [0, 1, 2, 3]
        assert r.top_indices[2].tolist() == [0, 1, 2, 3] and (r.top_logprobs[2, 1:] == -inf).all() and r.top_logprobs[2, 0] == 0
        assert r.entropy[2] == 0 and r.logprobs[2] == 0
        for row in (8, 9):
            assert torch.isnan(r.logprobs[row]) and torch.isnan(r.entropy[row]) and r.top_indices[row, 0] == 7
        index = top_of(x[ok], 4)[1]
        assert torch.equal(r.top_indices[ok], index)


@pytest.mark.parametrize("V", [90, 2500, 40000])
def test_ties_go_to_the_lowest_index(V):
    x = torch.zeros(4, V, device="cuda")
    x[1] = torch.randint(0, 3, (V,), device="cuda").float()
    x[2, V // 2:] = 1.0
    x[3, 5], x[3, 6] = 0.0, -0.0
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        check(x.to(dtype), t, top=32, grads=False)


def test_falling_and_rising_rows():
    """The best ones last, which replaces the list again and again, and first."""
    x = torch.arange(70000, device="cuda").float()[None] * 1e-3
    check(torch.cat([x, -x]), torch.tensor([3, 69999], device="cuda"), top=31)


def test_bad_targets_and_ignored_ones():
    from multi_gpu_flashattention_b200 import KernelStatusError, token_logprobs
    from multi_gpu_flashattention_b200.ops.flash import check_errors
    x = torch.randn(5, 600, device="cuda").requires_grad_()
    t = torch.tensor([3, 600, -1, -100, 7], device="cuda")
    r = token_logprobs(x, t)
    dx, = torch.autograd.grad([r.logprobs], [x], [torch.ones(5, device="cuda")])
    torch.cuda.synchronize()
    assert torch.isnan(r.logprobs[1:3]).all() and r.logprobs[3] == 0 and torch.isfinite(r.entropy).all()
    assert (dx[1:4] == 0).all() and (dx[[0, 4]] != 0).any()
    with pytest.raises(KernelStatusError, match="token_logprobs"):
        check_errors()
    # NaN gradients of ignored tokens count for nothing
    g = torch.tensor([1.0, 1.0, 1.0, float("nan"), 1.0], device="cuda")
    t = torch.tensor([3, 5, 6, -7, 7], device="cuda")
    r = token_logprobs(x, t, ignore_index=-7)
    dx, = torch.autograd.grad([r.logprobs], [x], [g])
    assert torch.isfinite(dx).all() and (dx[3] == 0).all()
    # an ignore_index that is a token
    r = token_logprobs(x, t.clamp(min=0), ignore_index=5)
    assert r.logprobs[1] == 0 and (r.logprobs[[0, 2, 4]] < 0).all()
    check_errors()


def test_no_rows_refusals_and_second_derivatives():
    from multi_gpu_flashattention_b200 import token_logprobs
    x, t = torch.randn(3, 50, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    empty = torch.randn(0, 50, device="cuda").requires_grad_()
    r = token_logprobs(empty, t[:0], top=3)
    assert r.logprobs.shape == (0,) and r.top_indices.shape == (0, 3)
    assert torch.autograd.grad(r.logprobs.sum(), empty)[0].shape == (0, 50)
    for match, args, kw in (("top must be", (x, t), dict(top=33)), ("top must be", (x, t), dict(top=-1)),
                            ("top must be", (x[:, :4], t), dict(top=5)), ("targets must have", (x, t[:2]), {}),
                            ("int32 or int64", (x, t.float()), {}), ("int32 or int64", (x, t.cpu()), {}),
                            ("bfloat16, float16 or float32", (x.double(), t), {}),
                            ("vocab", (x[:, :0], t), {})):
        with pytest.raises(RuntimeError, match=match):
            token_logprobs(*args, **kw)
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(token_logprobs(leaf, t).logprobs.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        g.sum().backward()
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            token_logprobs(fw.make_dual(x, torch.ones_like(x)), t)


def test_captured_steps_on_a_side_stream():
    from multi_gpu_flashattention_b200 import token_logprobs
    x = torch.randn(20, 20000, device="cuda", dtype=torch.bfloat16).requires_grad_()
    t = torch.randint(0, 20000, (20,), device="cuda")
    dl = torch.randn(20, device="cuda")

    def step():
        r = token_logprobs(x, t, top=6)
        return list(r) + list(torch.autograd.grad([r.logprobs, r.entropy], [x], [dl, dl]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
        t.copy_(torch.randint(0, 20000, (20,), device="cuda"))
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_large_offsets():
    """Rows that begin beyond 2^31 elements."""
    x = torch.zeros(17000, 131072, device="cuda", dtype=torch.bfloat16)
    x[-2:] = torch.randn(2, 131072, device="cuda").bfloat16()
    from multi_gpu_flashattention_b200 import token_logprobs
    t = torch.full((17000,), 131071, device="cuda")
    leaf = x.requires_grad_()
    r = token_logprobs(leaf, t, top=2)
    one = torch.ones(17000, device="cuda")
    dx, = torch.autograd.grad([r.logprobs], [leaf], [one])
    d = definition(x.detach()[-2:], t[-2:], one[-2:], 0 * one[-2:])
    close(r.logprobs[-2:], d["logprobs"], d["logprobs_err"])
    close(dx[-2:], d["dx"], d["dx_err"])
    assert torch.equal(r.top_indices[-2:], top_of(x.detach()[-2:], 2)[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [2000, 16000, 150000])
def test_alternatives_that_few_threads_hold(V, dtype):
    """All that is large lies in the vectors of `n` threads, more than is gathered at once; and in
    those of one thread."""
    per = 16 // torch.empty(0, dtype=dtype).element_size()
    threads = 32 if V < 2048 else 256
    lane = torch.arange(V, device="cuda") // per % threads
    x = torch.randn(8, V, device="cuda")
    for row, n in enumerate((1, 5, 15, 20, 31, 32, 64, 2)):
        x[row] += 20 * (lane < n) if row % 2 else 20 * (lane >= threads - n)
    t = torch.randint(0, V, (8,), device="cuda")
    for top in (1, 20, 32):
        check(x.to(dtype), t, top=top, grads=False)
