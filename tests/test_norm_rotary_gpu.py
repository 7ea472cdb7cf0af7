"""apply_norm_rotary and its gradients against the definition in 64 bits, and against
differences.

Tolerances, fixed before the first run, u = finfo.eps / 2 of the output's type, 2^-25 for
fp16's subnormals. A float32 step is 2^-24 = 6e-8. The sum of squares adds at most 16
squares a lane and 5 levels of lanes (element kernel: 8 and 5): 22 steps, half of which
reach rstd, with 3 of its own: 14 steps, 0.9e-6. Sine and cosine are off by 4e-7, the
products and sums of a rotation by 5 steps, the weights' by 2: 0.9e-6. So an output is off
by u|y| + 2e-6 (|n_a| + |n_b|) magnitude, and an angle t by 4 * 2^-53 |t| on top.
dx = rstd (g w - x^ mean(g w x^)): g has 0.7e-6 of G = (|dy_a| + |dy_b|) magnitude, the mean
22 steps more, rstd enters up to three times: 5e-6 of rstd (G |w| + |x^| mean(G |w| |x^|)).
dw sums g x^ in chains: in a thread, over the groups of a CTA (up to 256), over the CTAs.
At the sizes here a thread adds at most 64 terms, a CTA 256 groups and the CTAs 19 + 16:
355 steps, 2.2e-5, with 2e-6 of each term: 2.5e-5 of the sum of G |x^|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _turn(x, t, rd, interleaved, magnitude, sizes=False):
    """x [B, L, H, D] in 64 bits rotated by t [B, L, rd / 2]; sizes: |a| + |b| instead."""
    z, tail = x[..., :rd], x[..., rd:]
    a, b = (z[..., 0::2], z[..., 1::2]) if interleaved else (z[..., :rd // 2], z[..., rd // 2:])
    t = t[:, :, None, :]
    if sizes:
        u = v = (a.abs() + b.abs()) * magnitude
        tail = tail.abs()
    else:
        u, v = (a * t.cos() - b * t.sin()) * magnitude, (a * t.sin() + b * t.cos()) * magnitude
    put = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([put, tail], -1)


def reference(x, w, dy, pos, inv, eps, interleaved, magnitude):
    """y, dx, dw in 64 bits and the sizes that their errors go by."""
    x, w, dy = x.double(), w.double(), dy.double()
    rd, t = 2 * inv.numel(), pos.double()[..., None] * inv
    rstd = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    xh = x * rstd
    y = _turn(xh * w, t, rd, interleaved, magnitude)
    y_size = _turn(xh * w, t, rd, interleaved, magnitude, sizes=True)
    g = _turn(dy, -t, rd, interleaved, magnitude)
    g_size = _turn(dy, -t, rd, interleaved, magnitude, sizes=True)
    dx = rstd * (g * w - xh * (g * w * xh).mean(-1, keepdim=True))
    dx_size = rstd * (g_size * w.abs() + xh.abs() * (g_size * w.abs() * xh.abs()).mean(-1, keepdim=True))
    return dict(y=y, y_size=y_size, dx=dx, dx_size=dx_size, dw=(g * xh).sum((0, 1, 2)),
                dw_size=(g_size * xh.abs()).sum((0, 1, 2)))


def angle_error(pos, inv):
    return 4 * 2.0 ** -53 * pos.abs().max().item() * inv.max().item() if pos.numel() else 0.0


def close(got, ref, size, rel):
    u = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    bound = u * ref.abs() + rel * size + 2.0 ** -25
    assert (err <= bound).all(), ((err - bound).max().item(), err.max().item())


def _inputs(B, L, heads, D, dtype, wtype, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    mk = lambda h: (torch.randn(B, L, h, D, device="cuda", generator=g) * 1.5).to(dtype)
    w = [(1 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(wtype) for _ in heads]
    return [mk(h) for h in heads], w, [mk(h) for h in heads]


def check(xs, ws, dys, pos, inv, outs, grads, interleaved=False, magnitude=1.0, eps=1e-6):
    """outs: y of each; grads: (dx, dw) of each."""
    rows = pos.expand(xs[0].shape[:2])
    more = angle_error(pos, inv)
    for x, w, dy, y, (dx, dw) in zip(xs, ws, dys, outs, grads):
        r = reference(x, w, dy, rows, inv, eps, interleaved, magnitude)
        assert y.shape == x.shape == dx.shape and y.dtype == x.dtype == dx.dtype and dw.dtype == w.dtype
        close(y, r["y"], r["y_size"], 2e-6 + more)
        close(dx, r["dx"], r["dx_size"], 5e-6 + more)
        close(dw, r["dw"], r["dw_size"], 2.5e-5 + more)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L,H,Hk,D,rd", [(1, 1, 1, 1, 64, 64), (2, 33, 8, 2, 128, 128), (1, 61, 32, 8, 128, 64),
                                           (3, 5, 3, 1, 128, 50), (1, 700, 4, 4, 64, 2), (1, 9, 2, 1, 7, 6),
                                           (1, 17, 5, 5, 256, 256), (1, 21, 3, 2, 256, 16), (1, 40, 130, 70, 64, 32),
                                           (1, 2000, 8, 2, 64, 32), (1, 13, 1, 1, 8, 2), (2, 3, 2, 2, 2, 2)])
def test_forward_and_gradients(B, L, H, Hk, D, rd, dtype, interleaved):
    from multi_gpu_flashattention_b200 import apply_norm_rotary, rotary_frequencies
    wtype = torch.float32 if L % 2 else dtype
    xs, ws, dys = _inputs(B, L, (H, Hk), D, dtype, wtype, seed=L)
    inv, mag = rotary_frequencies(rd, scaling="ramp", factor=4.0, original_length=4096, device="cuda")
    pos = torch.randint(0, 1 << 20, (B, L), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    leaves = [t.clone().requires_grad_() for t in xs + ws]
    q, k, wq, wk = leaves
    outs = apply_norm_rotary(q, k, pos, inv, wq, wk, interleaved=interleaved, magnitude=mag)
    dq, dk, dwq, dwk = torch.autograd.grad(outs, leaves, dys)
    check(xs, ws, dys, pos, inv, outs, [(dq, dwq), (dk, dwk)], interleaved, mag)
    with torch.no_grad():  # the same without a graph
        for a, b in zip(outs, apply_norm_rotary(*xs, pos, inv, *ws, interleaved=interleaved, magnitude=mag)):
            assert torch.equal(a, b)


def test_strides_offsets_and_expanded_gradients():
    """Cuts of one projection, heads first, a start off a 16-byte boundary, columns apart,
    int32 positions of the batch, gradients that are expanded or strided."""
    from multi_gpu_flashattention_b200 import apply_norm_rotary, rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    pos = (torch.arange(40, device="cuda") * 3).int()
    dtype = torch.bfloat16
    _, ws, _ = _inputs(2, 1, (1, 1), 64, dtype, dtype, 3)
    base = torch.randn(2, 40, 6, 64, device="cuda").to(dtype)
    forms = [base, base.transpose(1, 2).contiguous().transpose(1, 2),
             torch.randn(2, 40, 6, 65, device="cuda").to(dtype)[..., 1:],
             torch.randn(2, 40, 64, 6, device="cuda").to(dtype).transpose(2, 3),
             torch.randn(1, 40, 6, 64, device="cuda").to(dtype).expand(2, 40, 6, 64)]
    one = torch.randn((), device="cuda").to(dtype)
    backs = [torch.randn(2, 40, 6, 64, device="cuda").to(dtype), one.expand(2, 40, 6, 64),
             torch.randn(2, 40, 6, 1, device="cuda").to(dtype).expand(2, 40, 6, 64),
             torch.randn(2, 40, 6, 68, device="cuda").to(dtype)[..., 4:]]
    for x in forms:
        for dy in backs:
            q, k = x[:, :, :4].detach().requires_grad_(), x[:, :, 4:].detach().requires_grad_()
            wq, wk = (w.clone().requires_grad_() for w in ws)
            outs = apply_norm_rotary(q, k, pos, inv, wq, wk)
            assert outs[0].is_contiguous() and outs[1].is_contiguous()
            gq, gk = dy[:, :, :4], dy[:, :, 4:]
            dq, dwq, dk, dwk = torch.autograd.grad(outs, [q, wq, k, wk], [gq, gk])
            check([q.detach(), k.detach()], ws, [gq, gk], pos, inv, [o.detach() for o in outs], [(dq, dwq), (dk, dwk)])
    # three dimensions, no batch
    a = apply_norm_rotary(base[1], None, pos, inv, ws[0], None)
    assert torch.equal(a, apply_norm_rotary(base, None, pos, inv, ws[0], None)[1])


def test_gradients_of_some_inputs():
    from multi_gpu_flashattention_b200 import apply_norm_rotary, rotary_frequencies
    xs, ws, dys = _inputs(1, 12, (4, 2), 64, torch.float32, torch.float32, 5)
    inv, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(12, device="cuda")
    leaves = [t.clone().requires_grad_() for t in xs + ws]
    q, k, wq, wk = leaves
    outs = apply_norm_rotary(q, k, pos, inv, wq, wk)
    all4 = torch.autograd.grad(outs, leaves, dys, retain_graph=True)
    # one output's gradient alone
    dk, dwk = torch.autograd.grad([outs[1]], [k, wk], [dys[1]], retain_graph=True)
    assert torch.equal(dk, all4[1]) and torch.equal(dwk, all4[3])
    none = torch.autograd.grad([outs[1]], [q, wq], [dys[1]], retain_graph=True, allow_unused=True)
    assert none == (None, None)
    # one input that needs one
    for i in range(4):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate(xs + ws)]
        o = apply_norm_rotary(args[0], args[1], pos, inv, args[2], args[3])
        got = torch.autograd.grad(o, [args[i]], dys, allow_unused=True)
        assert torch.equal(got[0], all4[i]), i
    # k absent
    o = apply_norm_rotary(q, None, pos, inv, wq, None)
    dq, dwq = torch.autograd.grad([o], [q, wq], [dys[0]])
    assert torch.equal(dq, all4[0])
    close(dwq, all4[2].double(), torch.ones_like(dwq).double(), 1e-4)


def test_gradients_against_differences():
    """Along a direction v, with h = 2^-6: (L(x + hv) - L(x - hv)) / 2h of the kernel's outputs
    in float32 differs from the definition's by the outputs' errors over h, and the
    definition's from its own gradient by what 64 bits show; dx, dw by their tolerances."""
    from multi_gpu_flashattention_b200 import apply_norm_rotary, rotary_frequencies
    (x,), (w,), (dy,) = _inputs(1, 30, (3,), 128, torch.float32, torch.float32, 7)
    inv, _ = rotary_frequencies(96, device="cuda")
    pos = torch.arange(30, device="cuda") * 11
    rows, h = pos.expand(1, 30), 2.0 ** -6
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = apply_norm_rotary(xl, None, pos, inv, wl, None)
    dx, dw = torch.autograd.grad([y], [xl, wl], [dy])
    r = reference(x, w, dy, rows, inv, 1e-6, False, 1.0)
    noise = ((2e-6 + 2.0 ** -24) * r["y_size"] * dy.double().abs()).sum() * 1.1
    for vx, vw in ((torch.randn_like(x), torch.zeros_like(w)), (torch.zeros_like(x), torch.randn_like(w))):
        ends = [(x + s * h * vx, w + s * h * vw) for s in (1, -1)]
        ours = [(apply_norm_rotary(a, None, pos, inv, b, None).double() * dy.double()).sum() for a, b in ends]
        exact = [(reference(a, b, dy, rows, inv, 1e-6, False, 1.0)["y"] * dy.double()).sum() for a, b in ends]
        ours, exact = (ours[0] - ours[1]) / (2 * h), (exact[0] - exact[1]) / (2 * h)
        along = (r["dx"] * vx).sum() + (r["dw"] * vw).sum()
        grad_error = ((5e-6 + 2.0 ** -24) * r["dx_size"] * vx.abs()).sum() + (2.5e-5 * r["dw_size"] * vw.abs()).sum()
        got = (dx.double() * vx).sum() + (dw.double() * vw).sum()
        # the ends are themselves rounded to float32: 2^-24 of each input through the gradient
        ends_error = 2.0 ** -24 * ((r["dx_size"] * x.abs()).sum() + (r["dw_size"] * w.abs()).sum()) / h
        assert (got - ours).abs() <= grad_error + noise / h + ends_error + (exact - along).abs()


def test_values_at_the_edges():
    """Rows of zeros, of tiny and of large values; a row with an infinity is its own alone."""
    from multi_gpu_flashattention_b200 import apply_norm_rotary, rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(6, device="cuda")
    x = torch.randn(6, 2, 64, device="cuda")
    x[0] = 0
    x[1] *= 1e-18
    x[2] *= 1e15
    x[3, 1, 5] = float("inf")
    x[4, 0, 9] = float("nan")
    w = torch.ones(64, device="cuda")
    leaf = x.clone().requires_grad_()
    y = apply_norm_rotary(leaf, None, pos, inv, w, None)
    dy = torch.randn_like(y)
    dx, = torch.autograd.grad([y], [leaf], [dy])
    ok = torch.ones(6, 2, dtype=torch.bool, device="cuda")
    ok[3, 1] = ok[4, 0] = False
    assert torch.isfinite(y[ok]).all() and torch.isfinite(dx[ok]).all()
    assert torch.isnan(y[~ok]).any(-1).all()
    r = reference(x[None], w, dy[None], pos[None], inv, 1e-6, False, 1.0)
    for got, name, rel in ((y, "y", 2e-6), (dx, "dx", 5e-6)):
        close(got[ok], r[name][0][ok], r[name + "_size"][0][ok], rel)
    assert (y[0] == 0).all()


def test_no_tokens_or_heads():
    from multi_gpu_flashattention_b200 import apply_norm_rotary, rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    w = torch.ones(64, device="cuda", requires_grad=True)
    q = torch.zeros(0, 4, 64, device="cuda", requires_grad=True)
    o = apply_norm_rotary(q, None, torch.arange(0, device="cuda"), inv, w, None)
    dq, dw = torch.autograd.grad([o], [q, w], [torch.zeros_like(o)])
    assert dq.shape == q.shape and (dw == 0).all()
    k = torch.randn(3, 0, 64, device="cuda")
    q = torch.randn(3, 2, 64, device="cuda")
    qo, ko = apply_norm_rotary(q, k, torch.arange(3, device="cuda"), inv, w.detach(), w.detach())
    assert ko.shape == k.shape and torch.equal(qo, apply_norm_rotary(q, None, torch.arange(3, device="cuda"), inv, w.detach(), None))


def test_again_gives_the_same_bits():
    from multi_gpu_flashattention_b200 import apply_norm_rotary, rotary_frequencies
    xs, ws, dys = _inputs(1, 1500, (8, 2), 128, torch.bfloat16, torch.bfloat16, 9)
    inv, _ = rotary_frequencies(128, device="cuda")
    pos = torch.arange(1500, device="cuda")
    leaves = [t.clone().requires_grad_() for t in xs + ws]
    q, k, wq, wk = leaves
    seen = None
    for _ in range(3):
        now = torch.autograd.grad(apply_norm_rotary(q, k, pos, inv, wq, wk), leaves, dys)
        assert seen is None or all(torch.equal(a, b) for a, b in zip(now, seen))
        seen = now


def test_refusals():
    from multi_gpu_flashattention_b200 import apply_norm_rotary, rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    q = torch.randn(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    k, pos, w = q[:, :1], torch.arange(4, device="cuda"), torch.ones(64, device="cuda")
    ok = dict(q=q, k=k, positions=pos, inv_freq=inv, q_weight=w, k_weight=w)

    def refused(match, **change):
        with pytest.raises(RuntimeError, match=match):
            apply_norm_rotary(**{**ok, **change})

    apply_norm_rotary(**ok)
    refused("come together", k=None)
    refused("come together", k_weight=None)
    refused("must be a CUDA tensor \\[head_dim\\]", q_weight=w[:32])
    refused("must be a CUDA tensor \\[head_dim\\]", k_weight=w.cpu())
    refused("q's dtype or be float32", q_weight=w.half())
    refused("must have one dtype", q_weight=w.bfloat16())
    refused("eps must not be negative", eps=-1.0)
    refused("k must match q", k=k.half())
    refused("inv_freq has", q=q[..., :32], k=k[..., :32], q_weight=w[:32], k_weight=w[:32])
    refused("positions must be", positions=pos[:3])
    refused("bfloat16, float16 or float32", q=q.double(), k=k.double())
    refused("head_dim must be 2 to 256", q=torch.randn(4, 2, 300, device="cuda"))
    a = q.float().requires_grad_()
    y = apply_norm_rotary(a, None, pos, inv, w, None)
    g, = torch.autograd.grad([y], [a], [torch.ones_like(y)], create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        g.sum().backward()
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            apply_norm_rotary(fw.make_dual(q.float(), torch.ones_like(q.float())), None, pos, inv, w, None)


def test_captured_training_step():
    """Forward and gradients in one graph, on a side stream, replayed with other inputs."""
    from multi_gpu_flashattention_b200 import apply_norm_rotary, rotary_frequencies
    xs, ws, dys = _inputs(1, 70, (4, 2), 64, torch.bfloat16, torch.float32, 11)
    inv, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(70, device="cuda")
    leaves = [t.clone().requires_grad_() for t in xs + ws]

    def step():
        outs = apply_norm_rotary(leaves[0], leaves[1], pos, inv, leaves[2], leaves[3])
        return list(outs) + list(torch.autograd.grad(outs, leaves, dys))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    new, _, _ = _inputs(1, 70, (4, 2), 64, torch.bfloat16, torch.float32, 12)
    with torch.no_grad():
        for a, b in zip(leaves, new):
            a.copy_(b)
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
