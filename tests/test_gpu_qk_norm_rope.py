"""Norm and rotation of queries and keys (d2p_amd.qk_norm_rope) against the 64-bit form.

Tolerances: everything is computed in 32 bits and rounded once, so a result is within
u |y| (u the type's unit roundoff) plus 16 roundings of 2^-24 of the row's norm; the weights'
gradients, sums of N rows' products in 32 bits, within 2^-24 (64 + N^0.5) sum |terms|.
"""
import pytest
import torch

import _encoderref as ref
import d2p_amd

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def inputs(seed, B, L, Hq, Hkv, D, R, dtype, dev, rows=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q, k, gq, gk = (r(B, L, H, D).to(dtype).to(dev) for H in (Hq, Hkv, Hq, Hkv))
    wq, wk = ((1 + 0.3 * r(D)).to(dev) for _ in range(2))
    cos, sin = d2p_amd.rope_tables(rows or max(L, 1), R, device=dev)
    return q, k, gq, gk, wq, wk, cos, sin


def run(q, k, gq, gk, wq, wk, cos, sin, positions=None, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk) if t is not None]
    it = iter(leaves[2:])
    a = [leaves[0], leaves[1], next(it) if wq is not None else None, next(it) if wk is not None else None]
    oq, ok = d2p_amd.qk_norm_rope(*a, cos, sin, positions, **kw)
    grads = torch.autograd.grad((oq, ok), leaves, (gq, gk))
    return [oq.detach(), ok.detach(), *grads]


def check(q, k, gq, gk, wq, wk, cos, sin, positions=None, eps=1e-6, interleaved=False):
    got = run(q, k, gq, gk, wq, wk, cos, sin, positions, eps=eps, interleaved=interleaved)
    u = ref.U[q.dtype]
    dws = iter(got[4:])
    for n, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        y, dx, dw = ref.norm_rope(x, w, cos, sin, positions, eps, interleaved, g)
        for have, want in ((got[n], y), (got[2 + n], dx)):
            bound = u * want.abs() + 16 * 2.0 ** -24 * want.norm(dim=-1, keepdim=True) + 1e-30
            err = (have.cpu().double() - want).abs()
            if n >= 0 and have is got[2 + n]:
                # dx is a difference of two terms of the gradient's size
                r = 1 / torch.sqrt((x.cpu().double() ** 2).mean(-1, keepdim=True) + eps)
                wm = 1.0 if w is None else float(w.abs().max())
                bound = bound + 32 * 2.0 ** -24 * r * wm * g.cpu().double().norm(dim=-1, keepdim=True)
            assert (err <= bound).all(), (n, float((err / bound).max()))
        if w is not None:
            _, _, terms = ref.norm_rope(x.abs(), None, cos * 0 + 1, sin * 0, positions, eps,
                                        interleaved, g.abs())
            # |rotated gradient| <= |a| + |c|: twice the terms without rotation, over pairs
            _, _, swapped = ref.norm_rope(x.abs(), None, cos * 0, sin * 0 + 1, positions, eps,
                                          interleaved, g.abs())
            N = x.numel() // x.shape[-1]
            bound = 2.0 ** -24 * (64 + N ** 0.5) * (terms + swapped.abs() + terms.max()) + 1e-30
            err = (next(dws).cpu().double() - dw).abs()
            assert (err <= bound).all(), (n, float((err / bound).max()))


SIZES = [(1, 1, 1, 1, 8, 8), (2, 5, 3, 1, 16, 4), (1, 33, 4, 2, 32, 32), (2, 17, 2, 2, 40, 24),
         (3, 50, 8, 2, 64, 64), (1, 70, 2, 1, 80, 80), (1, 9, 4, 4, 96, 64), (2, 64, 6, 3, 128, 128),
         (1, 12, 2, 2, 128, 6), (1, 12, 2, 1, 72, 70), (2, 8, 2, 2, 64, 0), (1, 300, 1, 1, 24, 12)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes_and_types(cuda, size, dtype):
    for interleaved in (False, True):
        check(*inputs(1, *size, dtype, cuda), interleaved=interleaved)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_positions_and_no_weights(cuda, dtype):
    q, k, gq, gk, wq, wk, cos, sin = inputs(2, 3, 20, 4, 2, 64, 32, dtype, cuda, rows=500)
    at = torch.randint(0, 500, (3, 20), generator=torch.Generator().manual_seed(3),
                       dtype=torch.int32).to(cuda)
    check(q, k, gq, gk, wq, wk, cos, sin, at)
    check(q, k, gq, gk, None, wk, cos, sin, at, eps=1e-3)
    # positions of another type and shape; one the table does not have
    want = d2p_amd.qk_norm_rope(q, k, wq, wk, cos, sin, at[:1].expand(3, 20).contiguous())
    got = d2p_amd.qk_norm_rope(q, k, wq, wk, cos, sin, at[0].long())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for wrong in (-1, 500, 2 ** 31):
        far = at.long()
        far[1, 7] = wrong
        oq, ok = d2p_amd.qk_norm_rope(q, k, wq, wk, cos, sin, far)
        for o in (oq, ok):
            nan = torch.isnan(o[..., :32])
            assert nan[1, 7].all() and nan.sum() == nan[1, 7].numel()
    plain = d2p_amd.qk_norm_rope(q, k, wq, wk)
    still = d2p_amd.qk_norm_rope(q, k, wq, wk, cos, sin, torch.zeros_like(at))
    assert all(torch.allclose(a.float(), b.float(), rtol=1e-6, atol=1e-6) for a, b in zip(plain, still))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(cuda, dtype):
    B, L, Hq, Hkv, D = 2, 40, 4, 2, 64
    q, k, gq, gk, wq, wk, cos, sin = inputs(4, B, L, Hq, Hkv, D, D, dtype, cuda)
    want = run(q, k, gq, gk, wq, wk, cos, sin)

    def same(a, b):
        # the weights' sums may run in another order where runs are narrower
        for n, (x, y) in enumerate(zip(a, b)):
            if n < 4:
                assert torch.allclose(x.float(), y.float(), rtol=2 * ref.U[x.dtype], atol=1e-6), n
            else:
                assert torch.allclose(x, y, rtol=1e-5, atol=1e-4), n

    qkv = torch.cat((q, k, k), 2)
    same(run(qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], gq, gk, wq, wk, cos, sin), want)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, gq, gk)]
    same(run(*heads_first, wq, wk, cos, sin), want)
    off = []
    for t in (q, k, gq, gk):
        flat = torch.zeros(t.numel() + 1, dtype=dtype, device=cuda)
        flat[1:] = t.flatten()
        off.append(flat[1:].view(t.shape))
    same(run(*off, wq, wk, cos, sin), want)
    apart = [t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0) for t in (q, k, gq, gk)]
    same(run(*apart, wq, wk, cos, sin), want)
    one = torch.ones((), dtype=dtype, device=cuda)
    same(run(q, k, one.expand(q.shape), one.expand(k.shape), wq, wk, cos, sin),
         run(q, k, torch.ones_like(q), torch.ones_like(k), wq, wk, cos, sin))


def test_one_result_used_and_same_bits(cuda):
    q, k, gq, gk, wq, wk, cos, sin = inputs(5, 4, 100, 8, 4, 64, 64, BF16, cuda)
    a = run(q, k, gq, gk, wq, wk, cos, sin)
    b = run(q, k, gq, gk, wq, wk, cos, sin)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    x, w = q.detach().requires_grad_(), wq.detach().requires_grad_()
    oq, _ = d2p_amd.qk_norm_rope(x, k, w, wk, cos, sin)
    dx, dw = torch.autograd.grad(oq, (x, w), gq)
    assert torch.equal(dx, a[2]) and torch.equal(dw, a[4])


def test_gradient_against_differences(cuda):
    """As for attention: a third of what doubling h changes, plus rounding."""
    args = inputs(6, 2, 11, 2, 1, 32, 24, F32, cuda)
    q, k, gq, gk, wq, wk, cos, sin = args
    got = run(*args)
    gen = torch.Generator().manual_seed(7)
    for n, x in enumerate((q, k, wq, wk)):
        d = torch.randn(x.shape, generator=gen).to(cuda)
        d = d / d.norm()

        def f(h):
            xs = [q, k, wq, wk]
            xs[n] = x + h * d
            oq, ok = d2p_amd.qk_norm_rope(*xs, cos, sin)
            return (oq.double() * gq).sum() + (ok.double() * gk).sum(), \
                (oq.double() * gq).abs().sum() + (ok.double() * gk).abs().sum()

        def diff(h):
            (a, s), (b, _) = f(h), f(-h)
            return (a - b) / (2 * h), 2.0 ** -22 * s / h

        fine, rounding = diff(0.125)
        coarse, _ = diff(0.25)
        want = (got[2 + n].double() * d.double()).sum()
        assert (fine - want).abs() <= (coarse - fine).abs() + 2 * rounding, (n, fine, want)


def test_refusals_and_empty(cuda):
    q, k, _, _, wq, wk, cos, sin = inputs(8, 2, 6, 4, 2, 32, 32, F32, cuda)
    f = d2p_amd.qk_norm_rope
    bad = [((q.double(), k, wq, wk, cos, sin), "float32, float16 or bfloat16"),
           ((q, k.to(BF16), wq, wk, cos, sin), "q's type"),
           ((q, k[:, :5], wq, wk, cos, sin), "same batch size, length"),
           ((q[..., :20], k[..., :20], None, None, None, None), "multiple of 8"),
           ((q, k, wq[:16], wk, cos, sin), "q_weight must be"),
           ((q, k, wq, wk, cos[:5], sin[:5]), "a row for each"),
           ((q, k, wq, wk, cos, sin[:, :4]), "both"),
           ((q, k, wq, wk, cos.to(F16), sin.to(F16)), "cos must be"),
           ((q, k, wq, wk, torch.ones(6, 17, device=cuda), torch.ones(6, 17, device=cuda)), "at most the head size"),
           ((q, k, wq, wk, cos, sin, torch.zeros(2, 5, dtype=torch.int32, device=cuda)), "positions must be"),
           ((q, k, wq, wk, cos, sin, torch.zeros(2, 6, device=cuda)), "positions must be"),
           ((q, k.cpu(), wq, wk, cos, sin), "CUDA tensor")]
    for args, match in bad:
        with pytest.raises(RuntimeError, match=match):
            f(*args)
    with pytest.raises(RuntimeError, match="eps"):
        f(q, k, eps=-1.0)
    with pytest.raises(RuntimeError, match="gradients"):
        f(q.requires_grad_(), k, wq, wk, cos.requires_grad_(), sin)
    with pytest.raises(ValueError, match="together"):
        f(q, k, wq, wk, cos)
    for B, L in ((0, 4), (2, 0)):
        args = inputs(9, B, L, 2, 2, 16, 16, BF16, cuda, rows=4)
        got = run(*args)
        assert got[0].shape == (B, L, 2, 16) and all((x == 0).all() for x in got)
