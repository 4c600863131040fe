"""SequenceAttention and the example that trains with it: the layer against the same layer
of elementary torch operations in 64 bits, its cache, torch.compile, the alignment on top.
"""
import importlib.util
import os

import pytest
import torch

import d2p_amd

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location(
        "train_encoder", os.path.join(ROOT, "examples", "train_encoder.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_layer(m, x, lengths, causal):
    """The layer's forward in 64 bits, differentiable."""
    B, L, _ = x.shape
    Hq, Hkv, D = m["heads"], m["kv"], m["D"]
    qkv = (x @ m["qkv"].T).view(B, L, Hq + 2 * Hkv, D)
    q, k, v = qkv.split((Hq, Hkv, Hkv), 2)

    def turn(t, w):
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
        a, b = t[..., :D // 2], t[..., D // 2:]
        c, s = m["cos"][:L, None], m["sin"][:L, None]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    q, k = turn(q, m["qn"]), turn(k, m["kn"])
    k, v = (t.repeat_interleave(Hq // Hkv, 2) for t in (k, v))
    i, j = torch.arange(L)[:, None], torch.arange(L)[None]
    R = m["buckets"].numel() // 2
    s = torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5
    s = s + m["bias"][m["buckets"].long()[(j - i).clamp(-R, R) + R]].permute(2, 0, 1)
    seen = (j < lengths[:, None, None]) & (i < lengths[:, None, None])
    if causal:
        seen = seen & (j <= i)
    s = s.masked_fill(~seen[:, None], -float("inf"))
    p = torch.softmax(s, -1).masked_fill(~seen[:, None], 0.0)
    return torch.einsum("bhij,bjhd->bihd", p, v).flatten(2) @ m["out"].T


@pytest.mark.parametrize("causal", [False, True])
def test_layer_against_plain(cuda, causal):
    """float32 throughout: six products and a softmax of values near 1, within 2e-5 of the
    largest (2^-24 times sums of up to 128 terms in each of them)."""
    torch.manual_seed(1)
    layer = d2p_amd.SequenceAttention(96, 6, 2, causal=causal, num_buckets=16, max_distance=20).to(cuda)
    torch.nn.init.normal_(layer.bias)
    torch.nn.init.normal_(layer.q_norm, 1.0, 0.2)
    x = torch.randn(3, 50, 96, device=cuda, requires_grad=True)
    lengths = torch.tensor([50, 17, 1], device=cuda)
    g = torch.randn(3, 50, 96, device=cuda)
    got = layer(x, lengths)
    names = ("qkv", "out", "qn", "kn", "bias")
    params = (layer.qkv.weight, layer.out.weight, layer.q_norm, layer.k_norm, layer.bias)
    grads = torch.autograd.grad(got, (x, *params), g)
    m = {n: p.detach().cpu().double().requires_grad_() for n, p in zip(names, params)}
    m.update(heads=6, kv=2, D=16, cos=layer.cos.cpu().double(), sin=layer.sin.cpu().double(),
             buckets=layer.buckets.cpu())
    xd = x.detach().cpu().double().requires_grad_()
    want = plain_layer(m, xd, lengths.cpu(), causal)
    wants = torch.autograd.grad(want, (xd, *(m[n] for n in names)), g.cpu().double())
    for a, b in zip((got.detach(), *grads), (want.detach(), *wants)):
        assert (a.cpu().double() - b).abs().max() <= 2e-5 * b.abs().max()


def test_layer_drops_in_training_only(cuda):
    torch.manual_seed(2)
    layer = d2p_amd.SequenceAttention(64, 2, dropout=0.3).to(cuda)
    x = torch.randn(2, 40, 64, device=cuda)
    a, b = layer(x, seed=5), layer(x, seed=5)
    assert torch.equal(a, b) and not torch.equal(a, layer(x, seed=6))
    torch.manual_seed(3)
    c = layer(x)
    torch.manual_seed(3)
    assert torch.equal(c, layer(x)) and not torch.equal(c, layer(x))
    layer.eval()
    assert torch.equal(layer(x), layer(x))


def test_cache_gives_what_the_whole_sequence_gives(cuda):
    """float32: the same sums in another order, 1e-5 of values near 1."""
    assert example().stream(report=lambda _: None) <= 1e-5
    torch.manual_seed(4)
    layer = d2p_amd.SequenceAttention(64, 4, causal=True).to(cuda).eval()
    x = torch.randn(2, 30, 64, device=cuda)
    cache = layer.new_cache(2, 40)
    whole = layer(x)
    parts = torch.cat([layer.step(x[:, a:b], cache) for a, b in ((0, 7), (7, 8), (8, 30))], 1)
    assert (whole - parts).abs().max() <= 1e-5 and cache.lengths.tolist() == [30, 30]


def test_a_full_cache_says_so(cuda):
    torch.manual_seed(6)
    layer = d2p_amd.SequenceAttention(64, 4, causal=True).to(cuda).eval()
    x = torch.randn(2, 6, 64, device=cuda)
    cache = layer.new_cache(2, 8, torch.bfloat16)
    cache.lengths.copy_(torch.tensor([0, 5], device=cuda))
    first = layer.step(x[:, :3], cache)
    assert first.dtype == torch.float32 and first.isfinite().all()
    second = layer.step(x[:, :2], cache)          # the second sequence has no room left
    assert second[0].isfinite().all() and second[1].isnan().all()
    third = layer.step(x, cache)
    assert third.isnan().all()
    with pytest.raises(ValueError, match="do not fit"):
        layer.step(torch.randn(2, 9, 64, device=cuda), cache)
    with pytest.raises(ValueError, match="causal"):
        d2p_amd.SequenceAttention(64, 4).to(cuda).step(x, cache)


def test_layer_compiles(cuda):
    torch.manual_seed(5)
    layer = d2p_amd.SequenceAttention(64, 2, num_buckets=8, max_distance=16).to(cuda)
    x = torch.randn(2, 33, 64, device=cuda, requires_grad=True)
    f = torch.compile(lambda t: layer(t), backend="aot_eager", fullgraph=True)
    got, want = f(x), layer(x)
    assert torch.equal(got, want)
    g = torch.randn_like(got)
    assert torch.equal(torch.autograd.grad(got, x, g)[0], torch.autograd.grad(want, x, g)[0])


def test_example_learns(cuda):
    """Related pairs become the higher-valued: the loss of the last steps is below that of
    guessing (log 2) and of the first."""
    for autocast in (True, False):
        losses = example().train(steps=30, batch=16, length=64, autocast=autocast, report=lambda _: None)
        last = sum(losses[-5:]) / 5
        assert last < 0.6 and last < losses[0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_layer_in_16_bits(cuda, dtype):
    """A layer moved to 16 bits is its operators in 16 bits, with angles in 32."""
    torch.manual_seed(7)
    layer = d2p_amd.SequenceAttention(64, 4, 2, causal=True, num_buckets=8, max_distance=16)
    torch.nn.init.normal_(layer.bias)
    layer = layer.to(cuda).to(dtype).eval()
    x = torch.randn(2, 30, 64, device=cuda, dtype=dtype)
    q, k, v = layer.qkv(x).view(2, 30, 8, 16).split((4, 2, 2), 2)
    q, k = d2p_amd.qk_norm_rope(q, k, layer.q_norm, layer.k_norm,
                                *d2p_amd.rope_tables(30, 16, device=cuda))
    o = d2p_amd.attention(q, k, v, causal=True, bias=layer.bias, buckets=layer.buckets)
    got = layer(x)
    assert got.dtype == dtype and torch.equal(got, layer.out(o.flatten(2)))
    got.sum().backward()
    assert all(p.grad.dtype == dtype and p.grad.isfinite().all() for p in layer.parameters())
    cache = layer.new_cache(2, 30)
    assert cache.keys.dtype == dtype and layer.step(x, cache).isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_cache_of_another_type(cuda, dtype):
    """Tokens attend in the cache's type, with the bias's numbers as they are."""
    torch.manual_seed(8)
    layer = d2p_amd.SequenceAttention(64, 4, 2, causal=True, num_buckets=8, max_distance=16)
    torch.nn.init.normal_(layer.bias)
    layer = layer.to(cuda).to(dtype).eval()
    x = torch.randn(2, 9, 64, device=cuda, dtype=dtype)
    for of in (torch.float32, torch.float16, torch.bfloat16):
        cache = layer.new_cache(2, 9, of)
        got = layer.step(x, cache)
        q, k, v = layer._project(x, None)
        o = d2p_amd.attention(q.to(of), k.to(of), v.to(of), causal=True, bias=layer.bias.float(),
                              buckets=layer.buckets)
        assert got.dtype == dtype and torch.equal(got, layer.out(o.flatten(2).to(dtype)))


def test_lengths_below_zero_are_nan(cuda):
    """A cache whose lengths somebody made negative: that sequence is NaN, its neighbours are
    what they are without it, and nothing outside its own rows is written."""
    torch.manual_seed(9)
    layer = d2p_amd.SequenceAttention(64, 4, causal=True).to(cuda).eval()
    x = torch.randn(3, 2, 64, device=cuda)
    want_cache, cache = layer.new_cache(3, 8), layer.new_cache(3, 8)
    want = layer.step(x, want_cache)
    for wrong in (-1, -2, -7, -2 ** 31):
        cache = layer.new_cache(3, 8)
        cache.lengths[1] = wrong
        got = layer.step(x, cache)
        assert got[1].isnan().all(), wrong
        for b in (0, 2):
            assert torch.equal(got[b], want[b]) and torch.equal(cache.keys[b], want_cache.keys[b])
            assert torch.equal(cache.values[b], want_cache.values[b])


def test_cache_no_longer_than_the_tables(cuda):
    layer = d2p_amd.SequenceAttention(64, 4, causal=True, max_length=16).to(cuda).eval()
    with pytest.raises(ValueError, match="max_length"):
        layer.new_cache(2, 17)
    cache = layer.new_cache(2, 16)
    assert layer.step(torch.randn(2, 16, 64, device=cuda), cache).isfinite().all()
    longer = d2p_amd.KeyValueCache(*(torch.zeros(2, 17, 4, 16, device=cuda) for _ in range(2)),
                                   torch.zeros(2, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError, match="max_length"):
        layer.step(torch.randn(2, 1, 64, device=cuda), longer)
