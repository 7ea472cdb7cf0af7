"""apply_rotary and its gradient against the definition in 64 bits.

Tolerance, fixed before the first run: one rounding of the output (u = finfo.eps / 2,
and 2^-25 for fp16's subnormals), and 1e-6 of |a| + |b| times the magnitude for sine
and cosine (the reduced angle in 32 bits is off by pi 2^-24 = 2e-7, each function by 2
steps, 2e-7) and the two products (2e-7). An angle t in 64 bits is itself known to
2^-53 |t| a rounding only: one in the reference (position times frequency), three in
the kernel (that product, 1 / 2 pi, and its product), so 4 * 2^-53 |t| of |a| + |b| on
top, which counts from positions of 10^9 on.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _ref(x, pos, inv, interleaved, magnitude, sign=1.0):
    """x [B, L, H, D], pos [B, L] -> (rotated, |a| + |b|), both float64."""
    rd = 2 * inv.numel()
    z = x[..., :rd].double()
    a, b = (z[..., 0::2], z[..., 1::2]) if interleaved else (z[..., :rd // 2], z[..., rd // 2:])
    t = (pos.double()[..., None] * inv * sign)[:, :, None, :]
    ra, rb = (a * t.cos() - b * t.sin()) * magnitude, (a * t.sin() + b * t.cos()) * magnitude
    s = (a.abs() + b.abs()) * magnitude
    put = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if interleaved else \
        (lambda u, v: torch.cat([u, v], -1))
    tail = x[..., rd:].double()
    return torch.cat([put(ra, rb), tail], -1), torch.cat([put(s, s), tail.abs()], -1)


def _close(got, x, pos, inv, interleaved, magnitude, sign=1.0):
    ref, size = _ref(x, pos, inv, interleaved, magnitude, sign)
    u = torch.finfo(x.dtype).eps / 2
    err = (got.double() - ref).abs()
    assert got.shape == x.shape and got.dtype == x.dtype
    angle = 4 * 2.0 ** -53 * pos.abs().max().item() * inv.max().item()
    assert (err <= u * ref.abs() + (1e-6 + angle) * size + 2.0 ** -25).all(), err.max().item()
    rd = 2 * inv.numel()
    assert torch.equal(got[..., rd:], x[..., rd:])


def _inputs(B, L, H, Hk, D, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    mk = lambda h: torch.randn(B, L, h, D, device="cuda", generator=g).to(dtype)
    return mk(H), mk(Hk), mk(H), mk(Hk)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L,H,Hk,D,rd", [(1, 1, 1, 1, 64, 64), (2, 33, 8, 2, 128, 128), (1, 61, 32, 8, 128, 64),
                                           (3, 5, 3, 1, 128, 50), (1, 700, 4, 4, 64, 2), (1, 9, 2, 1, 7, 6),
                                           (1, 17, 5, 5, 256, 256), (1, 3000, 8, 2, 64, 32)])
def test_forward_and_gradient(B, L, H, Hk, D, rd, dtype, interleaved):
    from multi_gpu_flashattention_b200 import apply_rotary, rotary_frequencies
    q, k, dq, dk = _inputs(B, L, H, Hk, D, dtype, seed=L)
    inv, mag = rotary_frequencies(rd, scaling="ramp", factor=4.0, original_length=4096, device="cuda")
    g = torch.Generator("cuda").manual_seed(1)
    pos = torch.randint(0, 1 << 20, (B, L), device="cuda", generator=g)
    qs, ks = q.clone().requires_grad_(), k.clone().requires_grad_()
    qo, ko = apply_rotary(qs, ks, pos, inv, interleaved=interleaved, magnitude=mag)
    gq, gk = torch.autograd.grad([qo, ko], [qs, ks], [dq, dk])
    for got, x, s in ((qo, q, 1.0), (ko, k, 1.0), (gq, dq, -1.0), (gk, dk, -1.0)):
        _close(got, x, pos, inv, interleaved, mag, s)


@pytest.mark.parametrize("scaling", ["none", "linear", "base", "ramp"])
def test_far_positions_and_types_of_positions(scaling):
    from multi_gpu_flashattention_b200 import apply_rotary, rotary_frequencies
    q, k, _, _ = _inputs(1, 6, 2, 1, 128, torch.float32)
    inv, mag = rotary_frequencies(128, scaling=scaling, factor=8.0, original_length=8192, device="cuda")
    far = torch.tensor([[0, 1, -5, 131071, (1 << 31) - 1, -(1 << 31)]], device="cuda")
    for pos in (far, far.int()):
        qo, ko = apply_rotary(q, k, pos, inv, magnitude=mag)
        _close(qo, q, far, inv, False, mag)
        _close(ko, k, far, inv, False, mag)
    huge = far + (1 << 40)
    _close(apply_rotary(q, None, huge, inv), q, huge, inv, False, 1.0)


def test_layouts_strides_and_one_tensor():
    """[tokens, heads, dim], positions shared by the batch, cuts of one projection,
    heads first, a start off a 16-byte boundary."""
    from multi_gpu_flashattention_b200 import apply_rotary, rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(40, device="cuda") * 3
    rows = pos.expand(2, 40)
    both = torch.randn(2, 40, 6, 64, device="cuda").bfloat16()
    q, k = both[:, :, :4], both[:, :, 4:]
    qo, ko = apply_rotary(q, k, pos, inv)
    assert qo.is_contiguous() and ko.is_contiguous()
    _close(qo, q, rows, inv, False, 1.0)
    _close(ko, k, rows, inv, False, 1.0)
    assert torch.equal(apply_rotary(q[1], None, pos, inv), qo[1])
    heads_first = both.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(apply_rotary(heads_first, None, pos, inv), apply_rotary(both, None, pos, inv))
    off = torch.randn(2, 40, 6, 65, device="cuda").bfloat16()[..., 1:]
    _close(apply_rotary(off, None, pos, inv, interleaved=True), off, rows, inv, True, 1.0)
    last = torch.randn(2, 40, 64, 6, device="cuda").bfloat16().transpose(2, 3)
    _close(apply_rotary(last, None, pos, inv), last, rows, inv, False, 1.0)


def test_gradient_of_one_side_and_of_expanded_inputs():
    from multi_gpu_flashattention_b200 import apply_rotary, rotary_frequencies
    q, k, dq, dk = _inputs(1, 12, 4, 4, 64, torch.float32)
    inv, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(12, device="cuda")
    ks = k.clone().requires_grad_()
    _, ko = apply_rotary(q, ks, pos, inv)
    (gk,) = torch.autograd.grad([ko], [ks], [dk])
    _close(gk, dk, pos[None], inv, False, 1.0, -1.0)
    one = k[:, :, :1].clone().requires_grad_()  # one head shared by four
    _, ko = apply_rotary(q, one.expand(1, 12, 4, 64), pos, inv)
    (g1,) = torch.autograd.grad([ko], [one], [dk])
    torch.testing.assert_close(g1, gk.sum(2, keepdim=True), rtol=1e-5, atol=1e-5)


def test_gradient_against_differences():
    from multi_gpu_flashattention_b200 import apply_rotary, rotary_frequencies
    q, k, dq, dk = _inputs(1, 7, 2, 1, 32, torch.float32)
    inv, _ = rotary_frequencies(16, device="cuda")
    pos = torch.arange(7, device="cuda") * 11
    qs, ks = q.clone().requires_grad_(), k.clone().requires_grad_()
    grads = torch.autograd.grad(apply_rotary(qs, ks, pos, inv, magnitude=1.5), [qs, ks], [dq, dk])
    f = lambda a, b: sum((u.double() * v.double()).sum()
                         for u, v in zip(apply_rotary(a, b, pos, inv, magnitude=1.5), (dq, dk)))
    dirs = [torch.randn_like(q), torch.randn_like(k)]
    num = (f(q + dirs[0], k + dirs[1]) - f(q - dirs[0], k - dirs[1])) / 2  # linear: any step does
    ana = sum((g.double() * d.double()).sum() for g, d in zip(grads, dirs))
    assert abs(num - ana) < 1e-4 * (1 + abs(ana))


def test_empty_and_graph():
    from multi_gpu_flashattention_b200 import apply_rotary, rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    e = torch.empty(0, 4, 64, device="cuda")
    assert apply_rotary(e, e, torch.empty(0, dtype=torch.int64, device="cuda"), inv)[0].shape == e.shape
    q, k, _, _ = _inputs(1, 5, 2, 1, 64, torch.bfloat16)
    pos = torch.arange(5, device="cuda")
    apply_rotary(q, k, pos, inv)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = apply_rotary(q, k, pos, inv)
    pos.add_(1000)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, apply_rotary(q, k, pos, inv)))


def test_refusals():
    from multi_gpu_flashattention_b200 import apply_rotary, rotary_frequencies
    inv, _ = rotary_frequencies(64, device="cuda")
    q, k, _, _ = _inputs(2, 8, 2, 1, 64, torch.bfloat16)
    pos = torch.arange(8, device="cuda")
    for bad in (lambda: apply_rotary(q, k.half(), pos, inv), lambda: apply_rotary(q, k[:1], pos, inv),
                lambda: apply_rotary(q, k, pos[:7], inv), lambda: apply_rotary(q, k, pos.float(), inv),
                lambda: apply_rotary(q, k, pos, inv.float()), lambda: apply_rotary(q, k, pos.cpu(), inv),
                lambda: apply_rotary(q[..., :32], k[..., :32], pos, inv),
                lambda: apply_rotary(q.double(), k.double(), pos, inv),
                lambda: apply_rotary(q[0, 0], None, pos, inv)):
        with pytest.raises(RuntimeError):
            bad()
