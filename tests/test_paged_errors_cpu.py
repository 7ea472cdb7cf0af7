"""When the cache's calls raise what a kernel has reported: only where nothing is left half
done. The kernels are fakes that note their calls; the status word is on the host."""
import types

import pytest
import torch


@pytest.fixture
def cache(monkeypatch):
    from multi_gpu_flashattention_b200.ops import paged
    calls = []

    def kernel(name, result=None):
        return lambda *a: (calls.append(name), result)[1]

    fake = types.SimpleNamespace(
        cache_check=kernel("check"), cache_reserve=kernel("reserve", "positions"),
        cache_write=kernel("write"), cache_free=kernel("free"), cache_fork=kernel("fork"),
        cache_compact=kernel("compact"), paged_attention=kernel("attention", ("out", None)))
    monkeypatch.setattr(paged, "C", lambda: fake)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)
    k = torch.zeros(3, 4, 16, 1, 64, dtype=torch.bfloat16)
    c = paged.PagedKVCache(k, k.clone(), z(2, 4), z(2), z(4), z(2))
    calls.clear()
    c.calls = calls
    c._status.word.zero_()
    yield c
    c._status.word.zero_()


def _error(cache):
    cache._status.word[0] = 6 | 64 << 8  # too few free pages


def test_a_step_goes_on_behind_its_reserve(cache):
    """write() and attend() of the other sequences' layers run, whatever reserve() reported."""
    from multi_gpu_flashattention_b200 import KernelStatusError
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    assert cache.reserve([0, 1], [0, 1, 2], 2) == "positions"
    _error(cache)
    for layer in range(3):
        cache.write(layer, x, x, [0, 1], [0, 1, 2])
        assert cache.attend(layer, x, [0, 1], [0, 1, 2], 1) == "out"
    assert cache.calls == ["reserve"] + ["write", "attention"] * 3
    with pytest.raises(KernelStatusError, match="too few free pages"):
        cache.reserve([0, 1], [0, 1, 2], 2)
    assert cache.calls[-1] == "attention"  # it has reserved nothing
    assert cache.reserve([0, 1], [0, 1, 2], 2) == "positions"


@pytest.mark.parametrize("name,args", [("free", ([0],)), ("fork", ([0], [1])), ("compact", ())])
def test_an_earlier_error_skips_no_call(cache, name, args):
    """free(), fork() and compact() do their work and then raise it."""
    from multi_gpu_flashattention_b200 import KernelStatusError
    _error(cache)
    with pytest.raises(KernelStatusError, match="too few free pages"):
        getattr(cache, name)(*args)
    assert cache.calls == [name]
    getattr(cache, name)(*args)
    assert cache.calls == [name, name]


@pytest.mark.parametrize("layer", [-1, 3, 99])
def test_attend_takes_the_cache_s_layers_only(cache, layer):
    """As write() does: -1 is not the last layer."""
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(IndexError, match="not one of the cache's 3"):
        cache.attend(layer, x, [0], [0, 1], 1)
    assert cache.calls == []


def _lm(**kw):
    from multi_gpu_flashattention_b200 import RingTransformerLM
    a = dict(vocab=20, d_model=32, n_layers=2, n_heads=2, n_kv_heads=1, head_dim=64, mlp_mult=1)
    return RingTransformerLM(**dict(a, **kw)).to(torch.bfloat16)


@pytest.mark.parametrize("why", ["layers", "heads", "head_dim", "dtype", "ids", "max", "group"])
def test_serve_refuses_before_the_cache_grows(cache, why):
    """What would end the step in one of its layers, with the cache grown for it."""
    model, ids, most = _lm(), torch.zeros(2, dtype=torch.int64), 1
    if why == "layers":
        model = _lm(n_layers=4)  # the cache has 3
    elif why == "heads":
        model = _lm(n_kv_heads=2)
    elif why == "head_dim":
        model = _lm(head_dim=128)
    elif why == "dtype":
        model = _lm().float()
    elif why == "ids":
        ids = ids[None]
    elif why == "max":
        most = -1
    else:
        model = _lm(n_heads=129, d_model=16)
    with pytest.raises(ValueError):
        model.serve(ids, cache, torch.zeros(2, dtype=torch.int32), torch.arange(3, dtype=torch.int32), most)
    assert cache.calls == []
