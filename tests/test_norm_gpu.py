"""rms_norm, its gradients and its 8-bit output against the formulas in 64 bits.

Tolerances, fixed before the first run. u = finfo(dtype).eps / 2 is one rounding of an
output; the fp32 arithmetic before it is good to 2e-5 of the size of its terms (a sum
of up to 16384 squares in a tree of chains of at most 64, a square root and three
products); 2^-25 is half a step of fp16's subnormals.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-6
F32 = 2e-5
SUB = 2.0 ** -25


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _make(rows, dim, dtype, residual, seed=0, wdtype=None):
    g = torch.Generator("cuda").manual_seed(seed)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
    w = (1 + 0.3 * torch.randn(dim, device="cuda", generator=g)).to(wdtype or dtype)
    return mk(rows, dim), w, mk(rows, dim) if residual else None, mk(rows, dim), mk(rows, dim)


def _ref(x, w, r):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    hd = h.double()
    rstd = (hd.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return h, hd * rstd, rstd, hd * rstd * w.double()


def _within(got, ref, tol, what):
    bad = ((got.double() - ref).abs() > tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the tolerance, " \
        f"largest error {(got.double() - ref).abs().max().item()}"


def _check(x, w, r, dy, dh):
    from multi_gpu_flashattention_b200 import rms_norm
    dim, dtype = x.shape[-1], x.dtype
    xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
    rs = r.detach().requires_grad_() if r is not None else None
    h, n, rstd, y = _ref(x, w, r)
    tol_y = y.abs() * (_u(dtype) + F32) + SUB
    if r is None:
        got = rms_norm(xs, ws, eps=EPS)
        gx, gw = torch.autograd.grad([got], [xs, ws], [dy])
        up = torch.zeros_like(y)
    else:
        got, goth = rms_norm(xs, ws, residual=rs, eps=EPS)
        assert torch.equal(goth, h)
        gx, gr, gw = torch.autograd.grad([got, goth], [xs, rs, ws], [dy, dh])
        assert torch.equal(gx, gr)
        up = dh.double()
    assert got.shape == x.shape and gx.shape == x.shape and gw.dtype == w.dtype
    _within(got, y, tol_y, "y")
    with torch.no_grad():  # without a gradient: the same values
        plain = rms_norm(x, w, residual=r, eps=EPS)
    assert torch.equal(plain if r is None else plain[0], got)
    g = dy.double() * w.double()
    dot = (g * n).mean(-1, keepdim=True)
    size = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True)) + up.abs()
    dx = rstd * (g - n * dot) + up
    _within(gx, dx, dx.abs() * _u(dtype) + F32 * size + SUB, "dx")
    terms = (dy.double() * n).reshape(-1, dim)
    rows = terms.shape[0]
    _within(gw, terms.sum(0), terms.sum(0).abs() * _u(w.dtype) + SUB +
            ((64 + rows) * 2.0 ** -24 + F32) * terms.abs().sum(0), "dw")


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (5, 64), (1, 100), (257, 128), (33, 1000),
                                      (7, 1024), (700, 2056), (2, 4096), (1300, 4096), (3, 5001),
                                      (2, 8192), (3, 12345), (5, 16384), (9, 6806),
                                      (300, 30), (4, 10002)])
def test_forward_and_gradients(rows, dim, dtype, residual):
    _check(*_make(rows, dim, dtype, residual, seed=rows + dim))


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(2, 3), (3, 1), (4, 2), (9, 1), (7, 5), (17, 3), (6, 4), (5, 6)])
def test_rows_shorter_than_a_vector(rows, dim, dtype, residual):
    _check(*_make(rows, dim, dtype, residual, seed=rows + dim))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_weight(dtype):
    x, w, r, dy, dh = _make(130, 768, dtype, True, wdtype=torch.float32)
    _check(x, w, r, dy, dh)


def test_many_rows_of_few_columns():
    _check(*_make(40000, 40, torch.bfloat16, True))


@pytest.mark.parametrize("dim", [512, 500])
def test_strided_and_misaligned_inputs(dim):
    """Rows of a wider tensor, rows that start off a 16-byte boundary, a transposed
    tensor, an expanded gradient, a stack of dimensions."""
    x, w, r, dy, dh = _make(24, 2 * dim + 16, torch.bfloat16, True)
    cut = lambda t, o: t[:, o:o + dim]
    _check(cut(x, 0), w[:dim].clone(), cut(r, 8), cut(dy, 0), cut(dh, dim))
    _check(cut(x, 1), w[3:3 + dim], cut(r, 0), cut(dy, 5), cut(dh, 0))
    _check(cut(x, 0).t().contiguous().t(), w[:dim], cut(r, 0), cut(dy, 0), cut(dh, 0))
    _check(cut(x, 0), w[:dim], cut(r, 0), dy[:1, :dim].expand(24, dim), dh[:, :1].expand(24, dim))
    four = lambda t: cut(t, 0).contiguous().view(2, 3, 4, dim)
    _check(four(x), w[:dim], four(r), four(dy), four(dh))
    _check(four(x).transpose(0, 2), w[:dim], four(r).transpose(0, 2), four(dy).transpose(0, 2),
           four(dh).transpose(0, 2))


@pytest.mark.parametrize("dim", [4, 128, 1028, 4096, 8192])
def test_float32_rows_and_weights(dim):
    """Weights that are read in vectors, and those that are off their boundary."""
    x, w, r, dy, dh = _make(9, dim + 8, torch.float32, True, seed=dim)
    cut = lambda t, o: t[..., o:o + dim]
    for o in (0, 4, 1):
        _check(cut(x, 0), cut(w, o), cut(r, 4), cut(dy, 0), cut(dh, 8))
    _check(cut(x, 3), cut(w, 0), cut(r, 0), cut(dy, 0), cut(dh, 0))


@pytest.mark.parametrize("width", [9, 16, 33])
def test_rows_that_overlap(width):
    """A sliding window over one tensor: rows one element apart."""
    flat = torch.randn(400, device="cuda").bfloat16()
    x = flat.unfold(0, width, 1)
    _, w, r, dy, dh = _make(x.shape[0], width, torch.bfloat16, True)
    assert x.stride() == (1, 1)
    _check(x, w, r, dy, dh)


def test_gradients_that_do_not_arrive():
    """Only h used, only y used, only some inputs differentiable."""
    from multi_gpu_flashattention_b200 import rms_norm
    x, w, r, dy, dh = _make(9, 256, torch.float32, True)
    xs, ws, rs = (t.detach().requires_grad_() for t in (x, w, r))
    y, h = rms_norm(xs, ws, residual=rs)
    gx, gr, gw = torch.autograd.grad([h], [xs, rs, ws], [dh], retain_graph=True)
    assert torch.equal(gx, dh) and torch.equal(gr, dh) and not gw.any()
    a = torch.autograd.grad([y], [xs, rs, ws], [dy], retain_graph=True)
    b = torch.autograd.grad([y, h], [xs, rs, ws], [dy, torch.zeros_like(dh)])
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    y, h = rms_norm(x, ws, residual=r)
    (gw,) = torch.autograd.grad([y], [ws], [dy])
    assert torch.equal(gw, a[2])


def test_gradient_against_differences():
    from multi_gpu_flashattention_b200 import rms_norm
    x, w, r, dy, dh = _make(6, 96, torch.float32, True, seed=3)
    xs, ws, rs = (t.detach().requires_grad_() for t in (x, w, r))
    y, h = rms_norm(xs, ws, residual=rs)
    grads = torch.autograd.grad([y, h], [xs, ws, rs], [dy, dh])
    f = lambda a, b, c: sum((u.double() * v.double()).sum() for u, v in zip(rms_norm(a, b, residual=c), (dy, dh)))
    g = torch.Generator("cuda").manual_seed(5)
    for i in range(3):
        d = [torch.zeros_like(t) for t in (x, w, r)]
        d[i] = torch.randn(d[i].shape, device="cuda", generator=g)
        e = 2.0 ** -7
        num = (f(*(t + e * u for t, u in zip((x, w, r), d))) -
               f(*(t - e * u for t, u in zip((x, w, r), d)))) / (2 * e)
        ana = (grads[i].double() * d[i].double()).sum()
        # differences: e^2 in truth, 2^-24 * sqrt(values) / e in rounding, of terms of size 1
        assert abs(num - ana) < 2e-2 * (grads[i].norm() + 1)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,group", [(1, 16, 16), (5, 96, 32), (3, 64, 64), (130, 1024, 128),
                                            (8, 4096, 128), (2, 8192, 64), (3, 5120, 0), (7, 333, 0),
                                            (9, 16384, 0), (1, 1, 0), (300, 16384, 16)])
def test_eight_bits(rows, dim, group, dtype, residual):
    from multi_gpu_flashattention_b200 import rms_norm_fp8
    x, w, r, _, _ = _make(rows, dim, dtype, residual, seed=dim)
    if rows > 2:
        x[1] = 0  # a row of zeros (without a residual) has scale 1
    h, n, _, y = _ref(x, w, r)
    y8, scale, *rest = rms_norm_fp8(x, w, residual=r, eps=EPS, group=group)
    assert y8.dtype == torch.float8_e4m3fn and y8.shape == x.shape
    groups = dim // group if group else 1
    assert scale.shape == (rows, groups)
    if r is not None:
        assert torch.equal(rest[0], h)
    yg = y.view(rows, groups, -1)
    top = yg.abs().amax(-1)
    want = torch.where(top > 0, top / 448, torch.ones_like(top))
    _within(scale, want, F32 * want, "scale")
    got = y8.double().view(rows, groups, -1) * scale.double()[..., None]
    # e4m3 rounds by at most 2^-4 of the value, or half its smallest step, 2^-10 of the scale
    tol = torch.maximum(yg.abs() * 2.0 ** -4, 2.0 ** -10 * want[..., None]) + 2 * F32 * yg.abs()
    _within(got, yg, tol, "y8")


def test_eight_bits_of_misaligned_rows():
    from multi_gpu_flashattention_b200 import rms_norm_fp8
    x, w, r, _, _ = _make(20, 300, torch.bfloat16, True)
    for o, p in ((1, 0), (0, 3), (5, 5)):
        got = rms_norm_fp8(x[:, o:o + 256], w[p:p + 256], residual=r[:, p:p + 256], group=32)
        want = rms_norm_fp8(x[:, o:o + 256].clone(), w[p:p + 256].clone(),
                            residual=r[:, p:p + 256].clone(), group=32)
        for a, b in zip(got, want):
            assert torch.equal(a.float(), b.float())


def test_infinities_and_nan_stay_in_their_rows():
    from multi_gpu_flashattention_b200 import rms_norm, rms_norm_fp8
    x, w, _, _, _ = _make(6, 128, torch.float32, False)
    clean = rms_norm(x, w)
    x[1, 5], x[3, 7] = float("nan"), float("inf")
    y = rms_norm(x, w)
    y8, scale = rms_norm_fp8(x, w)
    for row in (0, 2, 4, 5):
        assert torch.equal(y[row], clean[row]) and torch.isfinite(y8[row].float()).all()
    assert y[1].isnan().all() and y8[1].float().isnan().all() and scale[1] == 1
    assert y[3, 7].isnan() and not y[3, :7].any()


def test_second_derivative_is_refused():
    from multi_gpu_flashattention_b200 import rms_norm
    x, w, _, dy, _ = _make(4, 64, torch.float32, False)
    xs = x.requires_grad_()
    (g,) = torch.autograd.grad([rms_norm(xs, w)], [xs], [dy], create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        g.sum().backward()


def test_training_step_in_a_graph():
    """Forward and gradients captured together, replayed on other values."""
    from multi_gpu_flashattention_b200 import rms_norm
    x, w, r, dy, dh = _make(70, 512, torch.bfloat16, True)
    xs, ws, rs = (t.requires_grad_() for t in (x, w, r))
    step = lambda: torch.autograd.grad(rms_norm(xs, ws, residual=rs), [xs, ws, rs], [dy, dh])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    with torch.no_grad():
        xs.mul_(2).add_(1)
    g.replay()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_empty():
    from multi_gpu_flashattention_b200 import rms_norm, rms_norm_fp8
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = rms_norm(x, w)
    gx, gw = torch.autograd.grad([y.sum()], [x, w])
    assert gx.shape == (0, 64) and not gw.any()
    with torch.no_grad():
        y8, scale = rms_norm_fp8(x, w, group=32)
    assert y8.shape == (0, 64) and scale.shape == (0, 2)


def test_side_stream_and_graph():
    from multi_gpu_flashattention_b200 import rms_norm
    x, w, r, dy, dh = _make(64, 1024, torch.bfloat16, True)
    want = rms_norm(x, w, residual=r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rms_norm(x, w, residual=r)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rms_norm(x, w, residual=r)
    x.copy_(dy)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, rms_norm(dy, w, residual=r)))


def test_gradients_do_not_depend_on_timing():
    from multi_gpu_flashattention_b200 import rms_norm
    x, w, _, dy, _ = _make(3000, 1024, torch.bfloat16, False)
    xs, ws = x.requires_grad_(), w.requires_grad_()
    runs = [torch.autograd.grad([rms_norm(xs, ws)], [xs, ws], [dy]) for _ in range(3)]
    for a, b in runs[1:]:
        assert torch.equal(a, runs[0][0]) and torch.equal(b, runs[0][1])


def test_refusals():
    from multi_gpu_flashattention_b200 import rms_norm, rms_norm_fp8
    x, w, r, _, _ = _make(4, 96, torch.bfloat16, True)
    for bad in (lambda: rms_norm(x, w[:64]), lambda: rms_norm(x, w.half()),
                lambda: rms_norm(x, w, residual=r.float()), lambda: rms_norm(x, w, residual=r[:2]),
                lambda: rms_norm(x.double(), w.double()), lambda: rms_norm(x, w.cpu()),
                lambda: rms_norm(x.cpu(), w), lambda: rms_norm(x, w, eps=-1.0),
                lambda: rms_norm(torch.zeros(2, 16385, device="cuda"), torch.zeros(16385, device="cuda")),
                lambda: rms_norm_fp8(x, w, group=64), lambda: rms_norm_fp8(x, w, group=48),
                lambda: rms_norm_fp8(x.requires_grad_(), w)):
        with pytest.raises(RuntimeError):
            bad()


def test_tangents_of_a_gradient_are_refused():
    import torch.autograd.forward_ad as fwd
    from multi_gpu_flashattention_b200 import rms_norm
    x, w, _, dy, _ = _make(4, 64, torch.float32, False)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            rms_norm(fwd.make_dual(x, dy), w)
        y = rms_norm(x.requires_grad_(), w)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.autograd.grad([y], [x], [fwd.make_dual(dy, dy)])
