"""residual_norm at the ends of float32's range: rows whose squares it does not hold, gates that
are infinite."""
import pytest
import torch

import d2p_amd

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
HUGE = 3e19         # squared, more than float32 holds


def rows(B, L, D, dtype, seed, cuda):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(B, L, D, generator=g).to(dtype).to(cuda)


def alternating(D, device):
    """No sum that float32 does not hold, but squares."""
    return HUGE * (1 - 2 * (torch.arange(D, device=device) % 2)).float()


def step(x, y, dh, dn, norm, post, w, b, pw, pb):
    """h, n and the gradients of x, y and the vectors that there are."""
    leaves = [t.detach().clone().requires_grad_() for t in (x, y, w, pw) if t is not None]
    it = iter(leaves)
    x, y, w, pw = (next(it) if t is not None else None for t in (x, y, w, pw))
    b, pb = (None if t is None else t.detach().clone().requires_grad_() for t in (b, pb))
    h, n = d2p_amd.residual_norm(x, y, w, b, norm=norm, post_norm=post, post_weight=pw, post_bias=pb)
    outs, grads = ((n,), (dn,)) if y is None else ((h, n), (dh, dn))
    leaves += [t for t in (b, pb) if t is not None]
    names = [k for k, t in zip(("x", "y", "w", "pw"), (x, y, w, pw)) if t is not None]
    names += [k for k, t in (("b", b), ("pb", pb)) if t is not None]
    got = dict(zip(names, torch.autograd.grad(outs, leaves, grads)))
    return h.detach(), n.detach(), got


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("D", [40, 512, 520, 2055])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_row_whose_squares_overflow_is_normed_to_zeros(cuda, dtype, D, norm):
    """1 / sqrt(infinity) is 0: the row's n is the bias, its own gradient that of h alone, and the
    vectors' gradients are what the other rows give."""
    w = torch.linspace(0.5, 1.5, D, device=cuda)
    b = torch.linspace(-1.0, 1.0, D, device=cuda) if norm == "layer" else None
    x, y = rows(2, 5, D, dtype, 1, cuda), rows(2, 5, D, dtype, 2, cuda)
    dh, dn = rows(2, 5, D, dtype, 3, cuda), rows(2, 5, D, dtype, 4, cuda)
    quiet = dn.clone()
    quiet[1, 2] = 0
    bad = x.clone()
    bad[1, 2] = alternating(D, cuda).to(dtype)
    rest = torch.ones(2, 5, dtype=torch.bool, device=cuda)
    rest[1, 2] = False
    for block in (None, y):
        h, n, got = step(bad, block, dh, dn, norm, None, w, b, None, None)
        h2, n2, want = step(x, block, dh, quiet, norm, None, w, b, None, None)
        zeros = torch.zeros(D, device=cuda) if b is None else b
        assert torch.equal(n[1, 2], zeros.to(dtype)) and torch.equal(n[rest], n2[rest])
        assert torch.equal(got["w"], want["w"]) and got["w"].isfinite().all()
        assert torch.equal(got["x"][rest], want["x"][rest])
        own = torch.zeros(D, dtype=dtype, device=cuda) if block is None else dh[1, 2]
        assert torch.equal(got["x"][1, 2], own)
        if block is not None:
            assert torch.equal(got["y"][1, 2], own) and torch.equal(h[rest], h2[rest])
        if b is not None:       # whose gradient has no part of x
            assert torch.equal(got["b"], step(x, block, dh, dn, norm, None, w, b, None, None)[2]["b"])


@pytest.mark.parametrize("post", ["rms", "layer"])
@pytest.mark.parametrize("D", [40, 520])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_block_whose_squares_overflow_joins_as_its_bias(cuda, dtype, D, post):
    w, pw = torch.linspace(0.5, 1.5, D, device=cuda), torch.linspace(1.5, 0.5, D, device=cuda)
    pb = torch.linspace(-1.0, 1.0, D, device=cuda) if post == "layer" else None
    x, y = rows(2, 5, D, dtype, 1, cuda), rows(2, 5, D, dtype, 2, cuda)
    dh, dn = rows(2, 5, D, dtype, 3, cuda), rows(2, 5, D, dtype, 4, cuda)
    bad = y.clone()
    bad[0, 4] = alternating(D, cuda).to(dtype)
    h, n, got = step(x, bad, dh, dn, "rms", post, w, None, pw, pb)
    want = x[0, 4].float() if pb is None else x[0, 4].float() + pb
    assert torch.equal(h[0, 4], want.to(dtype)) and n.isfinite().all()
    assert not got["y"][0, 4].any()
    assert all(t.isfinite().all() for t in got.values())
    # the weight's gradient: what it is without that row's part in the results' gradients
    dh[0, 4] = dn[0, 4] = 0
    quiet = step(x, y, dh, dn, "rms", post, w, None, pw, pb)[2]
    assert torch.equal(got["pw"], quiet["pw"])


def test_sums_that_overflow(cuda):
    """A mean that float32 does not hold makes its row NaN, and no other."""
    x = rows(1, 3, 72, F32, 5, cuda)
    n = d2p_amd.residual_norm(x, norm="layer")[1]
    x[0, 1] = 1e38
    got = d2p_amd.residual_norm(x, norm="layer")[1]
    assert got[0, 1].isnan().all() and torch.equal(got[0, ::2], n[0, ::2])


@pytest.mark.parametrize("post,bias", [(None, False), ("rms", False), ("rms", True), ("layer", False),
                                       ("layer", True)])
@pytest.mark.parametrize("kind", ["feature", "sequence", "token"])
def test_infinite_gates(cuda, kind, post, bias):
    """h as the formula in 64 bits has it: an infinite gate times z, NaN where z is 0."""
    B, L, D = 2, 3, 24
    for dtype, block in ((F32, F32), (F32, BF16), (BF16, BF16)):
        x, y = rows(B, L, D, dtype, 1, cuda), rows(B, L, D, block, 2, cuda)
        if not post:
            y[0, 0, :6] = 0
        w = pb = None
        if post:
            w = torch.linspace(-1.0, 1.0, D, device=cuda)
            if bias:        # larger than w v, and of either sign
                pb = 9.0 * (1 - 2 * (torch.arange(D, device=cuda) % 2)).float()
        gate = rows(B, L, D, F32, 3, cuda)
        gate = {"feature": gate[0, 0], "sequence": gate[:, :1], "token": gate}[kind].clone()
        for f, value in ((1, "inf"), (2, "-inf"), (4, "nan"), (7, "inf"), (12, "inf"), (23, "-inf")):
            gate[..., f] = float(value)
        h, _ = d2p_amd.residual_norm(x, y, norm=None, post_norm=post, post_weight=w, post_bias=pb,
                                     gate=gate, scale=0.5)
        z = y.double()
        if post:
            z = z - z.mean(-1, keepdim=True) if post == "layer" else z
            z = z / (z.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            z = z if pb is None else z + pb.double()
        want = x.double() + 0.5 * gate.double() * z
        assert torch.equal(h.isnan(), want.isnan()), (dtype, block)
        ends = want.isinf()
        assert ends.any() and torch.equal(h[ends].double(), want[ends])
        rest = ~ends & ~want.isnan()
        assert (h[rest].double() - want[rest]).abs().max() <= (2.0 ** -7 if dtype == BF16 else 1e-4) * 20
