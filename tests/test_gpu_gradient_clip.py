"""global_norm, clip_gradients and clip_grad_norm_ against sums in 64 bits."""
import pytest
import torch

import _stackref as ref
import d2p_amd

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = (F32, BF16, F16)


def tensors(sizes, seed=0, scale=0.1, types=TYPES):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(types[i % len(types)]) for i, n in enumerate(sizes)]


def close(got, want, bounds):
    for a, b, e in zip(got, want, bounds):
        assert ((a.detach().cpu().double() - b).abs() <= e).all()


LISTS = [(1,), (0, 3), (7, 8, 9, 1, 15), (8191, 8192, 8193), (3_000_001, 5, 70_000),
         tuple(range(1, 130)), tuple([3] * 128), tuple([5, 1000] * 140)]


@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)} of {sum(s)}")
def test_against_formulas(cuda, sizes):
    ts = tensors(sizes)
    dev = [t.to(cuda) for t in ts]
    keep = [t.clone() for t in dev]
    for ratio in (0.3, 0.999, 1.001, 5.0):
        _, _, norm = ref.clipped(ts, 1.0)
        want, bounds, _ = ref.clipped(ts, ratio * norm)
        got, n = d2p_amd.clip_gradients(dev, ratio * norm)
        assert n.dtype == F32 and n.shape == () and abs(float(n) - norm) <= 2.0 ** -23 * norm
        assert float(d2p_amd.global_norm(dev)) == float(n)
        close(got, want, bounds)
        assert all(torch.equal(a, b) for a, b in zip(dev, keep))
        if ratio > 1:
            assert all(torch.equal(a, b) for a, b in zip(got, dev))
        # into tensors that are there, and in place: the same
        out = [torch.full_like(t, 7.0) for t in dev]
        res, n2 = d2p_amd.clip_gradients(dev, ratio * norm, out=out)
        assert all(a is b for a, b in zip(res, out)) and float(n2) == float(n)
        same = [t.clone() for t in dev]
        versions = [t._version for t in same]
        d2p_amd.clip_gradients(same, ratio * norm, out=same)
        assert all(t._version > v for t, v in zip(same, versions))
        for a, b, c in zip(got, out, same):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_views_of_buffers(cuda):
    """Tensors that lie next to each other at any alignment: nothing between them is written."""
    for dtype in TYPES:
        base = torch.randn(50_000, generator=torch.Generator().manual_seed(3)).to(dtype).to(cuda)
        out = torch.full_like(base, 7.0)
        cuts = [(1, 2), (3, 10), (11, 19), (20, 8213), (8214, 20_000), (20_001, 49_999)]
        ts, os = [base[a:b] for a, b in cuts], [out[a:b] for a, b in cuts]
        d2p_amd.clip_gradients(ts, 1.0, out=os)
        want, bounds, _ = ref.clipped(ts, 1.0)
        close(os, want, bounds)
        rest = torch.ones(50_000, dtype=torch.bool)
        for a, b in cuts:
            rest[a:b] = False
        assert (out.cpu()[rest] == 7.0).all()


def test_parameters(cuda):
    torch.manual_seed(0)
    layer = torch.nn.Sequential(torch.nn.Linear(30, 50), torch.nn.Linear(50, 30, bias=False)).to(cuda)
    unused = torch.nn.Parameter(torch.zeros(3, device=cuda))
    layer(torch.randn(8, 30, device=cuda)).square().sum().backward()
    ps = [*layer.parameters(), unused, layer[0].weight]      # one of them twice
    grads = [p.grad.clone() for p in layer.parameters()]
    want, bounds, norm = ref.clipped(grads, 0.5)
    got = d2p_amd.clip_grad_norm_(iter(ps), 0.5)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm and unused.grad is None
    close([p.grad for p in layer.parameters()], want, bounds)
    again = float(d2p_amd.clip_grad_norm_(ps, 0.7))          # within: left as they are
    assert abs(again - 0.5) < 1e-6
    close([p.grad for p in layer.parameters()], want, bounds)
    alone = d2p_amd.clip_grad_norm_(layer[0].weight, 1e9)
    assert float(alone) == float(d2p_amd.global_norm([layer[0].weight.grad]))
    assert float(d2p_amd.clip_grad_norm_([unused], 1.0)) == 0.0


def test_values_at_the_ends(cuda):
    big = torch.full((1000,), 1e30, device=cuda)             # whose squares no float32 holds
    got, n = d2p_amd.clip_gradients([big], 1.0)
    assert abs(float(n) / (1e30 * 1000 ** 0.5) - 1) < 1e-6
    assert ((got[0] * 1000 ** 0.5 - 1).abs() < 1e-6).all()
    small = torch.full((1000,), 1e-30, device=cuda)
    assert abs(float(d2p_amd.global_norm([small])) / (1e-30 * 1000 ** 0.5) - 1) < 1e-6
    zero = torch.zeros(10, device=cuda)
    got, n = d2p_amd.clip_gradients([zero], 0.0)
    assert float(n) == 0.0 and not got[0].any()
    got, n = d2p_amd.clip_gradients([torch.ones(4, device=cuda)], 0.0)
    assert float(n) == 2.0 and not got[0].any()
    x = torch.ones(4, device=cuda)
    x[2] = float("inf")
    got, n = d2p_amd.clip_gradients([x], 1.0)
    assert float(n) == float("inf") and got[0].isnan().tolist() == [False, False, True, False]
    assert got[0][0] == 0
    got, n = d2p_amd.clip_gradients([x], float("inf"))
    assert torch.equal(got[0], x)
    x[1] = float("nan")
    got, n = d2p_amd.clip_gradients([x, zero], 1.0)
    assert n.isnan() and all(t.isnan().all() for t in got)
    x = torch.full((3,), 60000.0, dtype=F16, device=cuda)
    got, n = d2p_amd.clip_gradients([x], 1.0)
    assert ((got[0].float() * 3 ** 0.5 - 1).abs() <= 2.0 ** -11).all()


def test_orders_of_memory(cuda):
    """Dense memory in another order, strided tensors, broadcast sources."""
    a = torch.randn(40, 30, device=cuda)
    for t in (a.t(), a.view(2, 20, 30).permute(2, 0, 1), a[:, ::2], a[5:, 3:], a[:1].expand(9, 30)):
        want, bounds, norm = ref.clipped([t], 2.0)
        got, n = d2p_amd.clip_gradients([t], 2.0)
        assert got[0].shape == t.shape and abs(float(n) - norm) <= 2.0 ** -23 * norm
        close(got, want, bounds)
        for out in (torch.zeros(t.shape, device=cuda), torch.zeros(*t.shape, 2, device=cuda)[..., 0],
                    torch.zeros(t.t().shape if t.dim() == 2 else t.shape, device=cuda)):
            out = out if out.shape == t.shape else out.t()
            d2p_amd.clip_gradients([t], 2.0, out=[out])
            close([out], want, bounds)
    for t in (a.clone().t(), a.clone()[:, ::2]):             # in place
        want, bounds, _ = ref.clipped([t], 2.0)
        d2p_amd.clip_gradients([t], 2.0, out=[t])
        close([t], want, bounds)


def test_refusals(cuda):
    x, y = torch.ones(4, device=cuda), torch.ones(4, device=cuda)
    op = d2p_amd.clip_gradients
    for call, match in (
            (lambda: op([], 1.0), "at least one"), (lambda: op([x], -1.0), "max_norm"),
            (lambda: op([x], float("nan")), "max_norm"), (lambda: op([x.double()], 1.0), "float32, float16"),
            (lambda: op([x, y.cpu()], 1.0), "CUDA"), (lambda: op([x], 1.0, out=[]), "1 tensors"),
            (lambda: op([x], 1.0, out=[y[:2]]), "shapes"), (lambda: op([x], 1.0, out=[y.half()]), "shapes"),
            (lambda: op([x, x], 1.0, out=[x, x]), "share"), (lambda: op([x, y], 1.0, out=[y, x]), "share"),
            (lambda: op([x[:3]], 1.0, out=[x[1:]]), "share"),
            (lambda: op([x], 1.0, out=[y[:1].expand(4)]), "."),
            (lambda: d2p_amd.global_norm([]), "at least one")):
        with pytest.raises((RuntimeError, ValueError), match=match):
            call()
    assert torch.equal(x, torch.ones_like(x)) and torch.equal(y, x)
    z = torch.ones(4, device=cuda, requires_grad=True)
    for call in (lambda: op([z], 1.0), lambda: d2p_amd.global_norm([z]), lambda: op([x], 1.0, out=[z])):
        with pytest.raises(RuntimeError, match="derivative"):
            call()
    with torch.no_grad():
        assert float(d2p_amd.global_norm([z])) == 2.0
