"""token_embedding and its gradient against the formulas in 64 bits (tests/_stackref.py)."""
import pytest
import torch

import _stackref as ref
import d2p_amd

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def inputs(V, B, L, D, wtype, dtype, ragged, kind="mixed", seed=0, tokens=torch.int64):
    g = torch.Generator().manual_seed(seed)
    if kind == "mixed":         # a few frequent tokens among many
        t = (torch.rand(B, L, generator=g) ** 3 * V).long().clamp(max=V - 1)
        t = torch.randperm(V, generator=g)[t]
    elif kind == "one":
        t = torch.full((B, L), V // 2)
    elif kind == "falling":
        t = (V - 1 - torch.arange(B * L) % V).view(B, L)
    elif kind == "pairs":       # runs of many lengths, in order
        t = (torch.arange(B * L).double().sqrt().long() % V).view(B, L)
    w = torch.randn(V, D, generator=g).to(wtype)
    grad = torch.randn(B, L, D, generator=g).to(dtype)
    lengths = None
    if ragged:
        lengths = torch.randint(0, L + 1, (B,), generator=g).int()
        lengths[0] = L
    return t.to(tokens), w, grad, lengths


def check(t, w, grad, lengths, scale=1.0, padding=None, dtype=None, dev="cuda"):
    want, bound, dw, dbound = ref.embedding(t, w, lengths, scale, padding, dtype, grad)
    wd = w.to(dev).requires_grad_()
    got = d2p_amd.token_embedding(t.to(dev), wd, None if lengths is None else lengths.to(dev),
                                  scale=scale, padding=padding, dtype=dtype)
    assert got.dtype == (dtype or w.dtype) and got.shape == want.shape
    out = got.detach().cpu().double()
    assert torch.equal(out.isnan(), want.isnan())
    assert ((out - want).abs() <= bound)[~want.isnan()].all()
    gw, = torch.autograd.grad(got, wd, grad.to(dev))
    assert gw.dtype == w.dtype and gw.shape == w.shape
    off = (gw.cpu().double() - dw).abs()
    assert (off <= dbound).all(), float((off - dbound).max())
    again, = torch.autograd.grad(d2p_amd.token_embedding(
        t.to(dev), wd, None if lengths is None else lengths.to(dev), scale=scale, padding=padding,
        dtype=dtype), wd, grad.to(dev))
    assert torch.equal(gw, again)
    return gw


CASES = [
    # V, B, L, D, weight, out, ragged, tokens' kind
    (5, 1, 1, 8, F32, F32, False, "mixed"),
    (1, 2, 9, 11, F32, F32, False, "one"),
    (21, 3, 50, 64, F32, BF16, True, "mixed"),
    (4, 7, 333, 40, BF16, BF16, True, "mixed"),
    (64, 2, 700, 512, F16, F16, False, "mixed"),
    (65, 2, 701, 513, F32, F16, True, "mixed"),
    (300, 2, 700, 33, F16, F16, True, "mixed"),
    (70000, 1, 37, 16, BF16, BF16, False, "mixed"),
    (1000, 4, 3000, 24, F32, F32, True, "mixed"),
    (1000, 1, 8192, 24, BF16, BF16, False, "pairs"),
    (257, 1, 20000, 520, BF16, BF16, False, "mixed"),
    (65537, 3, 3001, 8, F32, BF16, True, "mixed"),
    (17, 1, 5000, 136, F32, F32, False, "one"),
    (900, 1, 40000, 9, F16, F16, False, "one"),
    (3000, 2, 5000, 72, BF16, BF16, False, "falling"),
    (500, 1, 30011, 200, F16, F16, False, "pairs"),
    (12, 2, 4096, 1100, F32, F32, True, "mixed"),
    (2, 1, 3, 2000, F32, BF16, False, "mixed"),
    # where one way of summing ends and the next begins
    (64, 3, 900, 192, BF16, BF16, True, "mixed"),
    (64, 3, 900, 193, BF16, BF16, True, "mixed"),
    (33, 2, 50, 9, F32, F16, False, "mixed"),
    (1, 1, 2000, 8, F16, F16, False, "mixed"),
    (1, 1, 700, 12289, F32, F32, False, "mixed"),
    (3000, 1, 1024, 40, BF16, BF16, False, "pairs"),
    (3000, 1, 1025, 40, BF16, BF16, False, "pairs"),
    (200, 1, 2048, 40, F32, F32, False, "falling"),
    (200, 1, 2049, 40, F32, F32, False, "falling"),
    (70000, 2, 2048, 16, F16, F16, True, "mixed"),
    (70000, 1, 4097, 16, F16, F16, False, "mixed"),
    (1100000, 1, 3000, 8, F32, F32, False, "mixed"),
    (5000, 1, 131072, 8, F32, F32, False, "mixed"),
    (5000, 1, 131073, 8, F32, F32, False, "falling"),
    (700, 3, 100001, 8, BF16, BF16, True, "pairs"),
    (3, 1, 7, 1 << 20, F32, BF16, False, "mixed"),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_formulas(cuda, case):
    V, B, L, D, wtype, dtype, ragged, kind = case
    for n, (tokens, padding, scale) in enumerate(((torch.int64, None, 1.0), (torch.int32, V // 2, D ** 0.5))):
        t, w, grad, lengths = inputs(V, B, L, D, wtype, dtype, ragged, kind, n, tokens)
        dw = check(t, w, grad, lengths, scale, padding, dtype)
        if padding is not None:
            assert not dw[padding].any()


def test_wrong_tokens_and_lengths(cuda):
    """They come back NaN and add nothing, the others are what they are without them."""
    t, w, grad, _ = inputs(50, 4, 30, 24, F32, F32, False)
    for tokens in (torch.int32, torch.int64):
        x = t.to(tokens).clone()
        x[0, 3], x[1, 0], x[2, 29], x[3, 5] = -1, 50, 2 ** 31 - 1, -2 ** 31
        check(x, w, grad, None)
        check(x, w, grad, None, padding=0)
        check(x, w, grad, torch.tensor([30, 0, 31, -1], dtype=torch.int32))
    x = t.clone()
    x[0, 0], x[1, 1] = 2 ** 40, -2 ** 40 + 3      # whose low 32 bits are tokens
    check(x, w, grad, None, padding=3)


def test_what_is_past_a_length_does_not_matter(cuda):
    t, w, grad, _ = inputs(50, 4, 30, 24, F32, F32, False)
    lengths = torch.tensor([30, 7, 0, 1], dtype=torch.int32)
    a = check(t, w, grad, lengths)
    past = torch.arange(30) >= lengths[:, None]
    t[past], grad[past] = -5, float("nan")
    assert torch.equal(a, check(t, w, grad.nan_to_num(0.0), lengths))
    wd = w.to(cuda).requires_grad_()
    out = d2p_amd.token_embedding(t.to(cuda), wd, lengths.to(cuda))
    assert not out[past.to(cuda)].any()
    assert torch.equal(a, torch.autograd.grad(out, wd, grad.to(cuda))[0])


def test_shapes_strides_and_empty_calls(cuda):
    t, w, grad, _ = inputs(50, 4, 30, 24, BF16, BF16, False)
    wd = w.to(cuda).requires_grad_()
    want = d2p_amd.token_embedding(t.to(cuda), wd)
    dwant, = torch.autograd.grad(want, wd, grad.to(cuda), retain_graph=True)
    # other shapes of the same tokens
    for shape in ((120,), (2, 2, 30), (4, 3, 10, 1)):
        got = d2p_amd.token_embedding(t.view(shape).to(cuda), wd)
        assert got.shape == (*shape, 24) and torch.equal(got.view_as(want), want)
        assert torch.equal(torch.autograd.grad(got, wd, grad.to(cuda).view(got.shape))[0], dwant)
    one = d2p_amd.token_embedding(t[0, 0].to(cuda), wd)
    assert one.shape == (24,) and torch.equal(one, want[0, 0])
    # transposed tokens and weights, gradients with strides of their own
    got = d2p_amd.token_embedding(t.t().contiguous().to(cuda).t(), wd)
    assert torch.equal(got, want)
    wt = w.t().contiguous().to(cuda).t().requires_grad_()
    got = d2p_amd.token_embedding(t.to(cuda), wt)
    assert torch.equal(got, want)
    for make in (lambda g: torch.cat((g, g), -1)[..., 24:], lambda g: torch.cat((g, g), 1)[:, :30],
                 lambda g: g.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda g: g.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda g: torch.cat((g.flatten()[:1], g.flatten()))[1:].view(g.shape)):
        assert torch.equal(torch.autograd.grad(want, wd, make(grad.to(cuda)), retain_graph=True)[0], dwant)
    broad = grad[:1, :1].to(cuda).expand(4, 30, 24)
    assert torch.equal(torch.autograd.grad(want, wd, broad, retain_graph=True)[0],
                       torch.autograd.grad(want, wd, broad.contiguous())[0])
    for shape in ((0,), (0, 5), (3, 0)):
        got = d2p_amd.token_embedding(torch.zeros(shape, dtype=torch.int64, device=cuda), wd)
        assert got.shape == (*shape, 24)
        assert not torch.autograd.grad(got.sum(), wd)[0].any()


def test_refusals(cuda):
    t, w = torch.zeros(2, 3, dtype=torch.int64, device=cuda), torch.zeros(5, 8, device=cuda)
    op = d2p_amd.token_embedding
    for call, match in (
            (lambda: op(t.float(), w), "int32 or int64"), (lambda: op(t, w.double()), "float32, float16"),
            (lambda: op(t, w[0]), "2D"), (lambda: op(t, w[:, :7]), "features"), (lambda: op(t, w[:0]), "rows"),
            (lambda: op(t, w.half(), dtype=torch.float32), "weight's type"),
            (lambda: op(t, w, torch.zeros(3, dtype=torch.int32, device=cuda)), "lengths must be"),
            (lambda: op(t, w, torch.zeros(2, dtype=torch.int64, device=cuda)), "lengths must be"),
            (lambda: op(t, w, torch.zeros(2, dtype=torch.int32)), "CUDA"),
            (lambda: op(t[0], w, torch.zeros(2, dtype=torch.int32, device=cuda)), "B, L"),
            (lambda: op(t, w, scale=float("inf")), "finite"), (lambda: op(t.cpu(), w), "CUDA|HIP")):
        with pytest.raises(RuntimeError, match=match):
            call()
    for padding in (5, -1):
        with pytest.raises(ValueError, match="padding"):
            op(t, w, padding=padding)
    x = op(t, w.requires_grad_()).sum()
    d, = torch.autograd.grad(x, w, create_graph=True)
    assert not d.requires_grad


def test_second_derivative_raises(cuda):
    t = torch.zeros(2, 3, dtype=torch.int64, device=cuda)
    w = torch.randn(5, 8, device=cuda, requires_grad=True)
    g = torch.randn(2, 3, 8, device=cuda, requires_grad=True)
    d, = torch.autograd.grad(d2p_amd.token_embedding(t, w), w, g, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(d.sum(), g)
