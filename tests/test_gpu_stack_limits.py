"""The operators around a sequence encoder's attention layers at the ends of their ranges: tensors
of more than 2^31 numbers, as many rows and sequences as there may be, and memory next to
what a call writes, through the C ABI."""
import ctypes

import pytest
import torch

import _capi
import d2p_amd
from test_stack_host import Embedding, Residual, Strides, Tensor, Vector, lib  # noqa: F401

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E = 2.0 ** -24
CODE = {F32: 0, F16: 1, BF16: 2}


@pytest.fixture
def clean(cuda):
    torch.cuda.empty_cache()
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


# 2^31 numbers and some more in 16 bits
L_WIDE, D_WIDE = 262_144 + 5, 8192


@pytest.mark.parametrize("V", [20, 50])
def test_embeddings_past_2_to_31_numbers(cuda, clean, V):
    g = torch.Generator().manual_seed(V)
    weight = torch.randn(V, D_WIDE, generator=g).to(BF16).to(cuda).requires_grad_()
    tokens = torch.randint(0, V - 1, (1, L_WIDE), generator=g).to(cuda)
    tokens[0, -3:] = V - 1          # that nothing else has
    out = d2p_amd.token_embedding(tokens, weight)
    rows = torch.tensor([0, L_WIDE // 2, 262_143, 262_144, L_WIDE - 1], device=cuda)
    assert torch.equal(out[0, rows], weight[tokens[0, rows]])
    grad = torch.zeros_like(out)
    grad[0, rows] = torch.randn(5, D_WIDE, generator=g).to(BF16).to(cuda)
    dw, = torch.autograd.grad(out, weight, grad)
    want = torch.zeros(V, D_WIDE, dtype=torch.float64, device=cuda)
    want.index_add_(0, tokens[0, rows], grad[0, rows].double())
    size = torch.zeros_like(want).index_add_(0, tokens[0, rows], grad[0, rows].double().abs())
    # five additions in 32 bits (of zeros otherwise), and the rounding of the sum
    assert ((dw.double() - want).abs() <= 5 * E * size + 2.0 ** -8 * want.abs() * 1.01).all()


@pytest.mark.parametrize("gate", [False, True])
def test_residual_rows_past_2_to_31_numbers(cuda, clean, gate):
    """The last rows give what they give in a tensor of their own."""
    g = torch.Generator().manual_seed(3)
    last = [torch.randn(1, 9, D_WIDE, generator=g).to(BF16).to(cuda) for _ in range(5)]
    w = torch.ones(D_WIDE, device=cuda)

    def wide(t):
        big = torch.zeros(1, L_WIDE, D_WIDE, dtype=BF16, device=cuda)
        big[:, -9:] = t
        return big

    def step(x, y, m, dh, dn):
        x, y, m = x.requires_grad_(), y.requires_grad_(), m.requires_grad_() if gate else None
        h, n = d2p_amd.residual_norm(x, y, w, norm="layer", post_norm="rms", gate=m)
        leaves = [x, y] + ([m] if gate else [])
        return [h.detach(), n.detach()] + list(torch.autograd.grad([h, n], leaves, [dh, dn]))

    want = step(*[t.clone() for t in last])
    got = step(*[wide(t) for t in last])
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert torch.equal(a[:, -9:], b)


def test_clipping_past_2_to_31_numbers(cuda, clean):
    t = torch.zeros(2 ** 31 + 8195, dtype=BF16, device=cuda)
    t[:3] = 2.0
    t[-3:] = 2.0
    small = torch.full((4,), 2.0, device=cuda)
    got, norm = d2p_amd.clip_gradients([t, small], 1.0, out=[t, small])
    # sqrt(10 * 4): 2 / sqrt(40) with the roundings of the factor, the product and the type
    assert abs(float(norm) - 40 ** 0.5) <= 40 ** 0.5 * 2.0 ** -23
    want = 2.0 / 40 ** 0.5
    ends = torch.cat([t[:3], t[-3:]]).double()
    assert ((ends - want).abs() <= want * (2.0 ** -8 + 4 * E)).all()
    assert ((small.double() - want).abs() <= want * 3 * E).all()
    assert not any(bool(part.any()) for part in t[3:-3].split(1 << 30))


@pytest.mark.parametrize("V", [32, 40])
def test_as_many_tokens_as_there_may_be(cuda, clean, V):
    N, D = 2 ** 31 - 1, 8
    tokens = torch.empty(1, N, dtype=torch.int32, device=cuda)
    want = torch.zeros(V, dtype=torch.float64)
    for part in tokens[0].split(1 << 28):
        torch.arange(part.numel(), out=part)
        part.remainder_(V - 1)
        n = part.numel()
        want[:V - 1] += torch.tensor([n // (V - 1) + (v < n % (V - 1)) for v in range(V - 1)])
    for n in (5, N // 2, *range(N - 7, N)):     # the last token: at both ends, and in between
        want[int(tokens[0, n])] -= 1
        want[V - 1] += 1
        tokens[0, n] = V - 1
    assert float(want.sum()) == N and want[V - 1] == 9
    grad = torch.ones(1, 1, D, dtype=BF16, device=cuda).expand(1, N, D)
    dw = torch.ops.d2p_amd.token_embedding_backward(grad, tokens, None, 1.0, -1, V, F32).cpu().double()
    # partial sums of at most 2^24 ones are exact, the others' joins are off by E of what there is
    assert torch.equal(dw[V - 1], torch.full((D,), 9.0, dtype=torch.float64))
    assert ((dw - want[:, None]).abs() <= want[:, None] * E * (N / V / 256)).all()
    assert torch.equal(dw, dw[:, :1].expand_as(dw))
    with pytest.raises(RuntimeError, match="must fit int32"):
        d2p_amd.token_embedding(tokens[:, :1].expand(1, N + 1), torch.ones(V, D, device=cuda))


def test_as_large_a_table_as_there_may_be(cuda, clean):
    V, D, N = 2 ** 31 - 2, 8, 5000
    weight = torch.zeros(V, D, dtype=BF16, device=cuda)
    g = torch.Generator().manual_seed(6)
    tokens = torch.randint(0, V, (1, N), generator=g).to(cuda)
    tokens[0, :40] = torch.arange(40, device=cuda) % 4 + V - 4
    tokens[0, 40:50] = 0
    rows = torch.unique(tokens)
    weight[rows] = torch.randn(len(rows), D, generator=g).to(BF16).to(cuda)
    assert torch.equal(d2p_amd.token_embedding(tokens, weight), weight[tokens])
    grad = torch.randint(-4, 5, (1, N, D), generator=g).to(BF16).to(cuda)
    del weight
    dw = torch.ops.d2p_amd.token_embedding_backward(grad, tokens, None, 1.0, -1, V, BF16)
    want = torch.zeros(len(rows), D, device=cuda).index_add_(
        0, torch.searchsorted(rows, tokens[0]), grad[0].float())
    assert torch.equal(dw[rows].float(), want)      # whole numbers up to 40 * 4 = 160: exact
    dw[rows] = 0
    assert not any(bool(part.any()) for part in dw.split(1 << 27))


def test_as_many_rows_as_there_may_be(cuda, clean):
    N, D = 2 ** 31 - 1, 8
    x, y = (torch.randn(1, 1, D, generator=torch.Generator().manual_seed(n)).to(BF16).to(cuda)
            for n in range(2))
    w = torch.ones(D, device=cuda)
    want = d2p_amd.residual_norm(x, y, w, norm="layer")
    got = d2p_amd.residual_norm(x.expand(1, N, D), y.expand(1, N, D), w, norm="layer")
    for a, b in zip(got, want):
        for part in a[0].split(1 << 28):
            assert bool((part == b[0]).all())


def test_more_sequences_than_a_launch_has_workgroups(cuda, clean):
    """A gate by sequence of four million sequences: each its own sum."""
    B, L, D = (1 << 22) + 77, 2, 8
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.zeros(B, L, D, dtype=BF16, device=cuda)
    y = torch.randint(-8, 9, (B, L, D), generator=g, device=cuda).to(BF16)
    dh = torch.randint(-8, 9, (B, L, D), generator=g, device=cuda).to(BF16)
    gate = torch.ones(B, 1, D, device=cuda, requires_grad=True)
    h, _ = d2p_amd.residual_norm(x, y, gate=gate, norm=None)
    assert torch.equal(h, y)
    got, = torch.autograd.grad(h, gate, dh)
    assert torch.equal(got, (y.float() * dh.float()).sum(1, keepdim=True))     # whole numbers


def test_a_long_list_in_a_graph(cuda):
    """More tensors than one launch takes; some listed twice as sources."""
    g = torch.Generator().manual_seed(5)
    ts = [torch.randn(3 + 37 * (i % 50), generator=g).to((F32, BF16, F16)[i % 3]).to(cuda)
          for i in range(400)]
    ts += ts[:5]
    fresh = [[torch.randn(t.numel(), generator=g).to(t.dtype).to(cuda) for t in ts[:400]]
             for _ in range(3)]
    d2p_amd.clip_gradients(ts, 2.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, norm = d2p_amd.clip_gradients(ts, 2.0)
        whole = d2p_amd.global_norm(ts)
    for new in fresh:
        for t, n in zip(ts, new):
            t.copy_(n)
        graph.replay()
        want, n = d2p_amd.clip_gradients(ts, 2.0)
        assert torch.equal(norm, n) and torch.equal(whole, n)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="share memory"):
        d2p_amd.clip_gradients(ts, 2.0, out=ts)


# ---------------------------------------------------------------------------
# memory next to what a call writes
# ---------------------------------------------------------------------------
class Guarded:
    """`numbers` of a type between two stretches of a pattern; `shift` elements off alignment."""
    ZONE = 1 << 14

    def __init__(self, numbers, dtype, fill=None, shift=0):
        size = torch.empty((), dtype=dtype).element_size()
        self.at, self.bytes = self.ZONE + shift * size, numbers * size
        self.raw = torch.full((2 * self.ZONE + self.bytes + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        self.inside = self.raw[self.at:self.at + self.bytes]
        if fill is not None:
            self.inside.copy_(fill.contiguous().reshape(-1).view(torch.uint8))
        self.before = self.raw.clone()

    @property
    def ptr(self):
        return ctypes.c_void_p(self.raw.data_ptr() + self.at)

    def whole(self):
        same = self.raw == self.before
        return bool(same[:self.at].all()) and bool(same[self.at + self.bytes:].all())

    def unchanged(self):
        return torch.equal(self.raw, self.before)


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("size", [(1, 1, 5, 8), (2, 37, 3, 11), (3, 50, 33, 9), (2, 700, 200, 77),
                                  (1, 9001, 1000, 24), (2, 6, 40, 515), (1, 3, 30, 1029)], ids=str)
@pytest.mark.parametrize("pair", [(F32, F32), (F32, F16), (BF16, BF16)], ids=str)
def test_embedding_writes_its_results_only(cuda, lib, size, pair):  # noqa: F811
    B, L, V, D = size
    g = torch.Generator().manual_seed(1)
    w = Guarded(V * D, pair[0], torch.randn(V, D, generator=g).to(pair[0]).to(cuda), 1)
    tokens = Guarded(B * L, torch.int64, torch.randint(0, V, (B, L), generator=g).to(cuda))
    grad = Guarded(B * L * D, pair[1], torch.randn(B * L, D, generator=g).to(pair[1]).to(cuda), 3)
    p = Embedding(CODE[pair[0]], CODE[pair[1]], B, L, V, D, tokens.ptr, 8, None, -1, 1.0,
                  Strides(L * D, D))
    out, dw = Guarded(B * L * D, pair[1], shift=1), Guarded(V * D, pair[0], shift=1)
    need = lib.d2p_token_embedding_backward_workspace_bytes(ctypes.byref(p))
    ws = Guarded(need, torch.uint8)
    assert lib.d2p_token_embedding(ctypes.byref(p), w.ptr, out.ptr, stream()) == 0
    assert lib.d2p_token_embedding_backward(ctypes.byref(p), grad.ptr, dw.ptr, ws.ptr, need,
                                            stream()) == 0
    torch.cuda.synchronize()
    assert all(t.whole() for t in (out, dw, ws))
    assert all(t.unchanged() for t in (w, tokens, grad))


@pytest.mark.parametrize("size", [(1, 1, 8), (2, 3, 11), (5, 7, 64), (3, 40, 77), (2, 5, 520),
                                  (2, 3, 1500), (1, 2, 8192)], ids=str)
@pytest.mark.parametrize("kind", [1, 2, 3], ids=["feature", "sequence", "token"])
@pytest.mark.parametrize("pair", [(F32, F32), (F32, F16), (BF16, BF16)], ids=str)
def test_residual_writes_its_results_only(cuda, lib, size, kind, pair):  # noqa: F811
    B, L, D = size
    g = torch.Generator().manual_seed(2)
    n = B * L * D

    def of(numbers, dtype, shift=0):
        return Guarded(numbers, dtype, torch.randn(numbers, generator=g).to(dtype).to(cuda), shift)

    x, dh = of(n, pair[0], 1), of(n, pair[0], 1)
    y, dn = of(n, pair[1], 1), of(n, pair[1], 1)
    vectors = [of(D, F32, 1) for _ in range(4)]
    gates = {1: D, 2: B * D, 3: n}[kind]
    gate = of(gates, pair[1], 1)
    rows = Strides(L * D, D)
    p = Residual(CODE[pair[0]], CODE[pair[1]], B, L, D, 1, rows, rows, rows, rows, 2, 2,
                 *[Vector(v.ptr, 0) for v in vectors], kind, gate.ptr, CODE[pair[1]],
                 {1: Strides(0, 0), 2: Strides(D, 0), 3: rows}[kind], 0.5, 0.7, 1e-5)
    h, out = Guarded(n, pair[0], shift=1), Guarded(n, pair[1], shift=1)
    stats = Guarded(4 * B * L, F32)
    assert lib.d2p_residual_norm(ctypes.byref(p), x.ptr, y.ptr, h.ptr, out.ptr, stats.ptr, stream()) == 0
    need = lib.d2p_residual_norm_backward_workspace_bytes(ctypes.byref(p))
    ws = Guarded(need, torch.uint8)
    dx, dy = Guarded(n, pair[0], shift=1), Guarded(n, pair[1], shift=1)
    dgate = Guarded(gates, pair[1], shift=1)
    dv = [Guarded(D, F32, shift=1) for _ in range(4)]
    stream_in = h if pair[0] == F32 else x
    assert lib.d2p_residual_norm_backward(
        ctypes.byref(p), dh.ptr, dn.ptr, stream_in.ptr, y.ptr, stats.ptr, dx.ptr, dy.ptr, dgate.ptr,
        *[v.ptr for v in dv], ws.ptr, need, stream()) == 0
    torch.cuda.synchronize()
    assert all(t.whole() for t in (h, out, stats, ws, dx, dy, dgate, *dv))
    assert all(t.unchanged() for t in (x, y, dh, dn, gate, *vectors))


def test_clipping_writes_its_results_only(cuda, lib):  # noqa: F811
    g = torch.Generator().manual_seed(4)
    sizes = [1, 7, 8, 9, 8191, 8192, 8193, 30_000] * 30
    types = [(F32, BF16, F16)[i % 3] for i in range(len(sizes))]
    src = [Guarded(n, t, torch.randn(n, generator=g).to(t).to(cuda), i % 5)
           for i, (n, t) in enumerate(zip(sizes, types))]
    dst = [Guarded(n, t, shift=i % 7) for i, (n, t) in enumerate(zip(sizes, types))]
    need = lib.d2p_global_norm_workspace_bytes(len(sizes))
    ws, norm = Guarded(need, torch.uint8), Guarded(1, F32)
    tensors = (Tensor * len(sizes))(*[Tensor(a.ptr, b.ptr, n, CODE[t])
                                      for a, b, n, t in zip(src, dst, sizes, types)])
    assert lib.d2p_clip_by_norm(tensors, len(sizes), 1.0, norm.ptr, ws.ptr, need, stream()) == 0
    torch.cuda.synchronize()
    assert all(t.whole() for t in (ws, norm, *dst)) and all(t.unchanged() for t in src)
    norm2 = Guarded(1, F32)
    assert lib.d2p_global_norm(tensors, len(sizes), norm2.ptr, ws.ptr, need, stream()) == 0
    torch.cuda.synchronize()
    assert ws.whole() and norm2.whole() and torch.equal(norm.inside, norm2.inside)
