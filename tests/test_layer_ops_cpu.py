"""Host-side parts of the decoder-layer operators: refusals of host tensors, and the
frequencies of rotary positions."""
import math

import pytest
import torch


def test_host_tensors_are_refused():
    from multi_gpu_flashattention_b200 import apply_rotary, rms_norm, rms_norm_fp8
    x, w = torch.randn(4, 64), torch.ones(64)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        rms_norm(x, w)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        rms_norm_fp8(x, w)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        apply_rotary(torch.randn(4, 2, 64), None, torch.arange(4), torch.ones(32, dtype=torch.float64))


def test_host_caches_are_refused():
    from multi_gpu_flashattention_b200 import PagedKVCache, paged_attention
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        PagedKVCache.allocate(1, 4, 16, 1, 64, 2, 64, device="cpu")
    i32 = dict(dtype=torch.int32)
    k = torch.zeros(4, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        paged_attention(k[0, :1], k, k, torch.zeros(1, 4, **i32), torch.ones(1, **i32),
                        torch.arange(2, **i32), 1)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_attention(k[0, :1].clone().requires_grad_(), k, k, torch.zeros(1, 4, **i32),
                        torch.ones(1, **i32), torch.arange(2, **i32), 1)


def test_gradient_of_the_8_bit_output_is_refused():
    from multi_gpu_flashattention_b200 import rms_norm_fp8
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_fp8(torch.randn(4, 64, requires_grad=True), torch.ones(64))


@pytest.mark.parametrize("rd", [2, 64, 128])
def test_frequencies(rd):
    from multi_gpu_flashattention_b200 import rotary_frequencies
    inv, mag = rotary_frequencies(rd)
    assert inv.dtype == torch.float64 and mag == 1.0
    for i in range(rd // 2):
        assert inv[i].item() == pytest.approx(10000.0 ** (-2 * i / rd), rel=1e-14)
    lin, _ = rotary_frequencies(rd, scaling="linear", factor=4.0)
    torch.testing.assert_close(lin * 4, inv)


def test_frequencies_by_base_and_by_frequency():
    from multi_gpu_flashattention_b200 import rotary_frequencies
    inv, _ = rotary_frequencies(128)
    wide, _ = rotary_frequencies(128, scaling="base", factor=8.0)
    assert wide[0] == 1.0 and wide[-1].item() == pytest.approx(inv[-1].item() / 8.0, rel=1e-12)
    ramp, mag = rotary_frequencies(128, scaling="ramp", factor=4.0, original_length=4096)
    turns = 4096 * inv / (2 * math.pi)
    assert mag == pytest.approx(1 + 0.1 * math.log(4.0))
    assert torch.equal(ramp[turns > 40], inv[turns > 40])
    torch.testing.assert_close(ramp[turns < 0.9], inv[turns < 0.9] / 4)
    share = ((inv - ramp) / (inv - inv / 4))[(turns < 30) & (turns > 1.2)]
    assert (share.diff() > 0).all() and share.min() > 0 and share.max() < 1


@pytest.mark.parametrize("kw", [dict(rotary_dim=63), dict(rotary_dim=0), dict(rotary_dim=64, base=1.0),
                                dict(rotary_dim=64, factor=0.5), dict(rotary_dim=64, scaling="other"),
                                dict(rotary_dim=64, scaling="ramp"), dict(rotary_dim=2, scaling="base")])
def test_frequencies_refused(kw):
    from multi_gpu_flashattention_b200 import rotary_frequencies
    with pytest.raises(ValueError):
        rotary_frequencies(**kw)


def test_frequencies_made_under_inference_mode_serve_training():
    from multi_gpu_flashattention_b200.models.transformer import _frequencies
    with torch.inference_mode():
        f = _frequencies(6, torch.device("cpu"))
    assert not f.is_inference()
    x = torch.ones(3, dtype=torch.float64, requires_grad=True)
    (x * f).sum().backward()  # saves f
    assert torch.equal(x.grad, f)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_reads_no_further_than_its_rows(dtype):
    """Shifted rows are read in the aligned 16-byte vectors that cover them, the very last
    row's last vector by elements: every other row's vectors have to end inside the tensor."""
    from multi_gpu_flashattention_b200._ext import C
    v = 128 // torch.finfo(dtype).bits
    shifted = set()
    for dim in range(1, 4 * v + 2):
        for rows in range(1, 2 * v + 2):
            for apart in (dim, dim + v):
                flat = torch.zeros((rows - 1) * apart + dim, dtype=dtype)
                assert flat.data_ptr() % 16 == 0
                x = flat.as_strided((rows, dim), (apart, 1))
                if C().norm_layout_of(x, torch.ones(dim, dtype=dtype), None) != 1:
                    continue
                shifted.add(dim)
                for r in range(rows - 1):
                    end = r * apart + dim
                    assert end + -end % v <= flat.numel(), (dim, rows, apart, r)
    assert {v - 1, v + 1, 2 * v - 1, 3 * v + 2} <= shifted  # the wider ones keep their vectors


def test_forward_mode_derivatives_are_refused():
    """They would be lost without a word."""
    import torch.autograd.forward_ad as fwd
    from multi_gpu_flashattention_b200 import apply_rotary, paged_attention, rms_norm, rms_norm_fp8
    x, w, f = torch.randn(4, 64), torch.ones(64), torch.ones(32, dtype=torch.float64)
    q, pos, i32 = torch.randn(4, 2, 64), torch.arange(4), dict(dtype=torch.int32)
    k = torch.zeros(4, 16, 1, 64, dtype=torch.bfloat16)
    ints = torch.zeros(1, 4, **i32), torch.ones(1, **i32), torch.arange(2, **i32), 1
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        calls = [lambda: rms_norm(dual(x), w), lambda: rms_norm(x, dual(w)),
                 lambda: rms_norm(x, w, residual=dual(x)), lambda: rms_norm_fp8(dual(x), w),
                 lambda: apply_rotary(dual(q), None, pos, f), lambda: apply_rotary(q, dual(q), pos, f),
                 lambda: apply_rotary(q, None, pos, dual(f)),
                 lambda: paged_attention(dual(k[0, :1]), k, k, *ints),
                 lambda: paged_attention(k[0, :1], k, dual(k), *ints)]
        for call in calls:
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
            with fwd._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="must be a CUDA tensor"):
                call()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: rms_norm(t, w), (x,), (x,))
