"""Normed query and key heads in the plain model (CPU), and host-side refusals of the operators
of sampling and training."""
import pytest
import torch
import torch.nn.functional as F


def _model(**kw):
    from multi_gpu_flashattention_b200 import RingTransformerLM
    torch.manual_seed(0)
    return RingTransformerLM(vocab=50, d_model=32, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=16, mlp_mult=2, **kw)


def test_the_plain_model_norms_the_heads():
    """The block against its formula, in float32: rounding of some hundred steps of 2^-24."""
    from multi_gpu_flashattention_b200 import RingLayout
    from multi_gpu_flashattention_b200.models import rotary
    m = _model(qk_norm=True)
    blk = m.blocks[0]
    torch.nn.init.normal_(blk.q_norm.weight, 1.0, 0.3)
    torch.nn.init.normal_(blk.k_norm.weight, 1.0, 0.3)
    x = torch.randn(1, 10, 32)
    lay = RingLayout("contiguous", 10, 1, mask="causal")
    got = blk(x, lay, backend="torch")
    norm = lambda t, w: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * w
    h = norm(x, blk.norm1.weight)
    q, k, v = (w(h).view(1, 10, -1, 16) for w in (blk.wq, blk.wk, blk.wv))
    pos = torch.arange(10)
    q, k = rotary(norm(q, blk.q_norm.weight), pos), rotary(norm(k, blk.k_norm.weight), pos)
    k, v = (t.repeat_interleave(2, 2) for t in (k, v))
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) / 4.0
    s = s.masked_fill(torch.ones(10, 10, dtype=torch.bool).triu(1), float("-inf"))
    a = torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v).reshape(1, 10, -1)
    y = x + blk.wo(a)
    y = y + blk.mlp(norm(y, blk.norm2.weight))
    torch.testing.assert_close(got, y, rtol=2e-5, atol=2e-5)


def test_parameters_and_flags():
    m, n = _model(), _model(qk_norm=True, fused_loss=True)
    assert not any("q_norm" in k for k in m.state_dict()) and not m.fused_loss
    assert n.state_dict()["blocks.1.k_norm.weight"].shape == (16,) and n.fused_loss
    # saved whole before the flags existed: the class's defaults
    for mod in (m, *m.blocks):
        mod.__dict__.pop("fused_loss", None), mod.__dict__.pop("qk_norm", None)
    ids = torch.randint(0, 50, (1, 12))
    from multi_gpu_flashattention_b200 import RingLayout
    lay = RingLayout("contiguous", 12, 1, mask="causal")
    loss = m.loss(ids, ids, lay, backend="torch")
    want = F.cross_entropy(m(ids, lay, backend="torch").flatten(0, 1), ids.flatten())
    torch.testing.assert_close(loss, want)


def test_the_loss_on_the_host_is_the_plain_one():
    from multi_gpu_flashattention_b200 import RingLayout
    ids = torch.randint(0, 50, (1, 12))
    lay = RingLayout("contiguous", 12, 1, mask="causal")
    a, b = _model(fused_loss=True), _model()
    assert torch.equal(a.loss(ids, ids, lay, backend="torch"), b.loss(ids, ids, lay, backend="torch"))


def test_host_tensors_are_refused():
    from multi_gpu_flashattention_b200 import apply_norm_rotary, shared_prefix, token_logprobs
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        apply_norm_rotary(torch.randn(4, 2, 64), None, torch.arange(4), torch.ones(32, dtype=torch.float64),
                          torch.ones(64), None)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        token_logprobs(torch.randn(4, 20), torch.zeros(4, dtype=torch.int64))
    i32 = dict(dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        shared_prefix(torch.zeros(2, 4, **i32), torch.ones(2, **i32), torch.arange(3, **i32), torch.tensor([0, 2], **i32), 16)


@pytest.mark.parametrize("qk_norm", [False, True])
def test_attention_gets_one_type_under_autocast(monkeypatch, qk_norm):
    """32-bit norm weights widen what products in 16 bits gave; q, k and v reach the attention alike."""
    from multi_gpu_flashattention_b200 import RingLayout
    from multi_gpu_flashattention_b200.models import transformer
    seen = []

    def attention(q, k, v, **kw):
        seen.append((q.dtype, k.dtype, v.dtype))
        return q

    monkeypatch.setattr(transformer, "ring_attention", attention)
    m = _model(qk_norm=qk_norm)
    with torch.autocast("cpu", torch.bfloat16):
        m(torch.randint(0, 50, (1, 10)), RingLayout("contiguous", 10, 1, mask="causal"))
    assert seen == [(torch.bfloat16,) * 3] * 2
    seen.clear()
    m(torch.randint(0, 50, (1, 10)), RingLayout("contiguous", 10, 1, mask="causal"))
    assert seen == [(torch.float32,) * 3] * 2


class _Cache:
    """Notes that a call has reached it."""

    def __init__(self, k):
        self.k, self.reserved = k, False

    def reserve(self, *a):
        self.reserved = True
        raise KeyError("reserved")


@pytest.mark.parametrize("cu_groups,fits", [
    (torch.tensor([0, 2]), False), (torch.tensor([[0, 2]], dtype=torch.int32), False),
    (torch.tensor([], dtype=torch.int32), False), (torch.tensor([0, 9, 2, 9], dtype=torch.int32)[::2], False),
    (torch.zeros(4096, dtype=torch.int32), False), (torch.zeros(2, dtype=torch.int32, device="meta"), False),
    (torch.zeros(4095, dtype=torch.int32), True), (torch.zeros(1, dtype=torch.int32), True),
    (torch.tensor([0, 2], dtype=torch.int32), True), ([0, 1, 2], True), ([], False), (None, True)])
def test_groups_are_refused_before_the_cache_grows(cu_groups, fits):
    m = _model()
    cache = _Cache(torch.zeros(2, 4, 16, 2, 16))
    slots, cu = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    with pytest.raises(KeyError if fits else ValueError, match="reserved" if fits else "cu_groups must be"):
        m.serve(torch.tensor([1, 2]), cache, slots, cu, 1, cu_groups=cu_groups)
    assert cache.reserved == fits


def test_norms_are_refused_before_the_cache_grows():
    def double(b):
        b.k_norm.double()

    def both(b):
        b.k_norm.double(), b.q_norm.double()

    def below(b):
        b.k_norm.eps = -1e-6

    slots, cu = torch.tensor([0], dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32)
    for change in (double, both, below, None):
        m = _model(qk_norm=True)
        if change:
            change(m.blocks[1])
        cache = _Cache(torch.zeros(2, 4, 16, 2, 16))
        with pytest.raises(ValueError if change else KeyError, match="heads' norms" if change else "reserved"):
            m.serve(torch.tensor([1, 2]), cache, slots, cu, 2)
        assert cache.reserved == (change is None)
