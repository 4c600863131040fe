"""Attention and its gradients (d2p_amd.attention) against the 64-bit form, within the
rounding bounds that tests/_encoderref.py derives; masks, strides, streams and graphs.
"""
import itertools

import pytest
import torch

import _encoderref as ref
import d2p_amd

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def inputs(seed, B, Lq, Lk, Hq, Hkv, D, dtype, dev, buckets=0, R=0, bias_type=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q, k, v, grad = (r(B, L, H, D).to(dtype).to(dev) for L, H in
                     ((Lq, Hq), (Lk, Hkv), (Lk, Hkv), (Lq, Hq)))
    bias = where = None
    if buckets:
        bias = r(buckets, Hq).to(bias_type or dtype).to(dev)
        where = torch.randint(0, buckets, (2 * R + 1,), generator=g, dtype=torch.int32).to(dev)
    return q, k, v, grad, bias, where


def run(q, k, v, grad=None, lengths=None, causal=False, scale=None, bias=None, buckets=None,
        drop=0, seed=0):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    if bias is not None:
        leaves.append(bias.detach().requires_grad_())
    b = leaves[3] if bias is not None else None
    out = d2p_amd.attention(*leaves[:3], lengths, causal=causal, scale=scale, bias=b,
                            buckets=buckets, dropout=drop / 256, seed=seed if drop else None)
    got = {"out": out.detach()}
    if grad is not None:
        got.update(zip(("dq", "dk", "dv", "dbias"), torch.autograd.grad(out, leaves, grad)))
    return got


def check(got, want, bounds):
    for n, x in got.items():
        x, y, e = x.cpu().double(), want[n], bounds[n]
        assert x.shape == y.shape and torch.isfinite(x).all(), n
        worst = ((x - y).abs() / (e + 1e-30)).max() if x.numel() else 0.0
        assert worst <= 1.0, (n, float(worst), float((x - y).abs().max()))


def both(args, grad=True, **kw):
    q, k, v, g, bias, where = args
    g = g if grad else None
    got = run(q, k, v, g, bias=bias, buckets=where, **kw)
    want = ref.attention(q, k, v, g, bias=bias, buckets=where, **kw)
    check(got, *want)
    return got


def lens(dev, *pairs):
    return torch.tensor(pairs, dtype=torch.int32, device=dev)


SIZES = [
    # B, Lq, Lk, Hq, Hkv, D
    (1, 1, 1, 1, 1, 8), (2, 1, 65, 4, 2, 32), (1, 2, 300, 2, 2, 64), (2, 33, 31, 2, 1, 40),
    (1, 64, 64, 2, 2, 128), (1, 129, 127, 3, 3, 80), (2, 200, 200, 4, 1, 64), (1, 65, 257, 2, 2, 96),
    (1, 300, 70, 1, 1, 128), (3, 100, 120, 2, 2, 32), (1, 7, 513, 8, 2, 16),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes_and_types(cuda, size, dtype):
    both(inputs(1, *size, dtype, cuda))
    both(inputs(2, *size, dtype, cuda), causal=True)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size,buckets,R", [((2, 70, 70, 2, 2, 64), 16, 32), ((1, 300, 300, 2, 1, 32), 32, 128),
                                            ((1, 130, 200, 2, 2, 128), 9, 5), ((2, 40, 50, 2, 2, 8), 3, 0),
                                            ((1, 150, 150, 1, 1, 64), 300, 1024), ((1, 70, 130, 2, 1, 128), 5, 1024),
                                             ((2, 90, 90, 2, 1, 96), 12, 40)], ids=str)
def test_bias_and_its_gradient(cuda, size, buckets, R, dtype):
    for causal, bias_type in ((False, dtype), (True, F32)):
        both(inputs(3, *size, dtype, cuda, buckets, R, bias_type), causal=causal)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size,drop,buckets", [((2, 70, 45, 4, 2, 32), 26, 0), ((1, 200, 200, 2, 2, 64), 128, 8),
                                               ((1, 66, 131, 2, 1, 128), 255, 0), ((2, 3, 300, 2, 1, 64), 51, 4)],
                         ids=str)
def test_dropout(cuda, size, drop, buckets, dtype):
    args = inputs(4, *size, dtype, cuda, buckets, 20)
    for causal in (False, True):
        both(args, causal=causal, drop=drop, seed=0x123456789abcdef)


def test_dropout_mask_is_the_generator_s(cuda):
    """Equal scores and one-hot values show the mask itself."""
    L, D = 128, 128
    z = torch.zeros(1, L, 2, D, device=cuda)
    v = torch.eye(D, device=cuda)[None, :, None].expand(1, L, 1, D)
    for seed in (0, 5, -1, 2 ** 63 + 11):
        out = d2p_amd.attention(z, z[:, :, :1], v, dropout=0.25, seed=seed)
        kept = (out[0] > 0).permute(1, 0, 2).cpu()
        assert torch.equal(kept, ref.keep_mask(1, 2, L, L, 64, seed)[0])
        t = torch.tensor([seed - 2 ** 64 if seed >= 2 ** 63 else seed], device=cuda)
        assert torch.equal(out, d2p_amd.attention(z, z[:, :, :1], v, dropout=0.25, seed=t))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("causal", [False, True])
def test_ragged_and_empty(cuda, dtype, causal):
    """Lengths down to nothing; more queries than keys, whose first rows see none; what lies
    past the lengths is NaN and infinity, and changes no bit."""
    ls = lens(cuda, (70, 90), (0, 40), (33, 0), (64, 64), (70, 13), (1, 1), (0, 0))
    args = inputs(5, len(ls), 70, 90, 4, 2, 64, dtype, cuda, 8, 16)
    got = both(args, lengths=ls, causal=causal, drop=32, seed=3)
    q, k, v, g, bias, where = (t.clone() for t in args)
    for b, (nq, nk) in enumerate(ls.tolist()):
        q[b, nq:] = float("nan")
        g[b, nq:] = float("inf")
        k[b, nk:] = float("-inf")
        v[b, nk:] = float("nan")
    again = run(q, k, v, g, ls, causal, None, bias, where, 32, 3)
    for n in got:
        assert torch.equal(got[n], again[n]), n
    if causal:
        assert (got["out"][4, :57] == 0).all() and (got["out"][4, 57:] != 0).any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_filled_card(cuda, dtype):
    """Enough blocks of queries for the wider workgroups that wide heads take then."""
    ls = lens(cuda, (520, 70), (257, 33), (1, 70), (519, 0))
    both(inputs(12, 4, 520, 70, 64, 4, 128, dtype, cuda), lengths=ls)
    both(inputs(13, 4, 520, 70, 64, 64, 128, dtype, cuda, 8, 16), causal=True, drop=40, seed=9)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_few_queries_use_nothing_past_the_lengths(cuda, D, dtype):
    ls = lens(cuda, (2, 3000), (1, 17), (2, 1), (2, 0), (0, 50), (1, 2049))
    q, k, v, _, bias, where = inputs(14, len(ls), 2, 3000, 4, 2, D, dtype, cuda, 8, 16)
    for causal in (False, True):
        want = run(q, k, v, None, ls, causal, None, bias, where)["out"]
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        for b, (nq, nk) in enumerate(ls.tolist()):
            q2[b, nq:] = float("inf")
            k2[b, nk:] = float("nan")
            v2[b, nk:] = float("-inf")
        assert torch.equal(run(q2, k2, v2, None, ls, causal, None, bias, where)["out"], want)
        assert (want[3] == 0).all() and (want[4] == 0).all() and want.isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_bias_that_masks(cuda, dtype):
    """-inf hides pairs, and a row of nothing else is zeros; the type's lowest value does not
    hide: rows of nothing else weigh their keys equally."""
    q, k, v, g, _, _ = inputs(6, 1, 40, 40, 2, 2, 32, dtype, cuda)
    where = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)   # behind, same place, ahead
    inf = torch.tensor([[0.5, -float("inf")], [-float("inf")] * 2, [-float("inf"), 1.0]]).to(dtype).to(cuda)
    args = (q, k, v, g, inf, where)
    got = run(q, k, v, g, bias=inf, buckets=where)
    check(got, *ref.attention(q, k, v, g, bias=inf, buckets=where))
    assert (got["out"][0, 0, 0] == 0).all() and (got["out"][0, -1, 1] == 0).all()
    low = torch.full((3, 2), torch.finfo(dtype).min, dtype=dtype, device=cuda)
    got = run(q, k, v, g, bias=low, buckets=where)
    mean = v.double().mean(1, keepdim=True).expand(1, 40, 2, 32)
    u = ref.U[dtype]
    assert ((got["out"].double() - mean).abs() <= 2 * u * v.double().abs().mean(1, keepdim=True) + 1e-5).all()
    want = g.double().sum(1, keepdim=True).expand(1, 40, 2, 32) / 40
    assert ((got["dv"].double() - want).abs() <= 2 * u * g.double().abs().mean(1, keepdim=True) + 1e-5).all()
    assert all(torch.isfinite(x).all() for x in got.values())
    del args


def test_wrong_numbers_on_the_device_are_nan(cuda):
    args = inputs(7, 3, 20, 30, 2, 2, 32, F32, cuda, 4, 3)
    ls = lens(cuda, (20, 30), (21, 30), (20, -1))
    got = run(*args[:4], ls, bias=args[4], buckets=args[5])
    for n in ("out", "dq", "dk", "dv"):
        assert torch.isfinite(got[n][0]).all() and torch.isnan(got[n][1:]).all(), n
    assert torch.isnan(got["dbias"]).any()
    where = args[5].clone()
    where[3] = 4                      # distance 0 in a bucket that does not exist
    assert torch.isnan(run(*args[:4], bias=args[4], buckets=where)["out"]).all()


def layouts(t):
    """The same values under other strides: packed with neighbours, heads first, misaligned,
    features apart."""
    B, L, H, D = t.shape
    packed = torch.zeros(B, L, 3 * H, D, dtype=t.dtype, device=t.device)
    packed[:, :, H:2 * H] = t
    yield packed[:, :, H:2 * H]
    yield t.transpose(1, 2).contiguous().transpose(1, 2)
    flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    yield flat[1:].view(t.shape)
    yield t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    wide = torch.zeros(B, L, H, D + 1, dtype=t.dtype, device=t.device)
    wide[..., :D] = t
    yield wide[..., :D]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(cuda, dtype):
    q, k, v, g, _, _ = inputs(8, 2, 50, 70, 4, 2, 40, dtype, cuda)
    want = run(q, k, v, g)
    for ql, kl, vl, gl in zip(layouts(q), layouts(k), layouts(v), layouts(g)):
        got = run(ql, kl, vl, gl)
        assert all(torch.equal(got[n], want[n]) for n in want)
    # one gradient value for all, one key for all of the batch, rows all the same
    ones = torch.ones((), dtype=dtype, device=cuda)
    same = run(q, k, v, ones.expand(q.shape))
    assert torch.equal(same["dq"], run(q, k, v, torch.ones_like(q))["dq"])
    kk = k[:1, :1].expand(k.shape).detach()
    assert torch.equal(run(q, kk, v)["out"], run(q, kk.contiguous(), v)["out"])
    shared = k[:1].clone().requires_grad_()
    out = d2p_amd.attention(q, shared.expand(k.shape), v)
    dk, = torch.autograd.grad(out, shared, g)
    full = run(q, shared.detach().expand(k.shape), v, g)["dk"]
    assert torch.equal(dk, full.sum(0, keepdim=True))


def test_offsets_past_32_bits(cuda):
    """Keys and values whose rows lie 128 KiB apart: the last at 9 GiB."""
    L, D = 70001, 64
    big = torch.zeros((L, 65536), dtype=BF16, device=cuda)
    q, k, v, _, _, _ = inputs(9, 1, 3, L, 2, 1, D, BF16, cuda)
    big[:, :D], big[:, D:2 * D] = k[0, :, 0], v[0, :, 0]
    kk, vv = big[None, :, None, :D], big[None, :, None, D:2 * D]
    for causal in (False, True):
        assert torch.equal(run(q, kk, vv, causal=causal)["out"], run(q, k, v, causal=causal)["out"])
    q = q[:, :1].expand(1, 130, 2, D).contiguous()
    assert torch.equal(run(q, kk, vv)["out"], run(q, k, v)["out"])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_token_of_a_long_cache(cuda, dtype):
    for size in ((3, 1, 5000, 8, 2, 64), (1, 4, 9001, 4, 1, 128), (2, 1, 2500, 2, 2, 40), (1, 9, 4000, 16, 2, 32)):
        both(inputs(10, *size, dtype, cuda, 8, 16), grad=False, causal=True)
    args = inputs(11, 4, 2, 6000, 4, 2, 64, dtype, cuda)
    both(args, grad=False, causal=True, lengths=lens(cuda, (2, 6000), (1, 17), (2, 1), (2, 0)))


def test_gradient_against_differences(cuda):
    """Directional derivatives of <out, g> by central differences of the kernel itself: the
    error of a difference at h is at most a third of what doubling h changes (truncation goes
    with h^2), plus the rounding of two results, 2^-22 sum |out g| / h."""
    q, k, v, g, bias, where = inputs(12, 2, 37, 53, 4, 2, 32, F32, cuda, 6, 9)
    drop = dict(drop=40, seed=99)
    got = run(q, k, v, g, bias=bias, buckets=where, **drop)
    gen = torch.Generator().manual_seed(13)
    names = ("dq", "dk", "dv", "dbias")
    for n, (name, x) in enumerate(zip(names, (q, k, v, bias))):
        d = torch.randn(x.shape, generator=gen).to(cuda)
        d = d / d.norm()

        def f(h):
            xs = [q, k, v, bias]
            xs[n] = x + h * d
            out = run(*xs[:3], bias=xs[3], buckets=where, **drop)["out"].double()
            return (out * g.double()).sum(), (out * g.double()).abs().sum()

        def diff(h):
            (a, s), (b, _) = f(h), f(-h)
            return (a - b) / (2 * h), 2.0 ** -22 * s / h

        fine, rounding = diff(0.125)
        coarse, _ = diff(0.25)
        want = (got[name].double() * d.double()).sum()
        assert (fine - want).abs() <= (coarse - fine).abs() + 2 * rounding, (name, fine, want)


@pytest.mark.parametrize("group", [1, 2])
def test_small_and_uneven_gradients_in_half(cuda, group):
    """Gradients of a millionth, one head's a thousand times another's, one head's zero:
    powers of two between them, so the relative bounds hold as they stand."""
    q, k, v, g, _, _ = inputs(20, 2, 90, 110, 4, 4 // group, 64, F16, cuda)
    g = g * torch.tensor([2.0 ** -14, 2.0 ** -4, 0.0, 2.0 ** -10], device=cuda)[:, None]
    got = run(q, k, v, g.half())
    check(got, *ref.attention(q, k, v, g.half()))
    big = run(q, k, v, torch.full_like(q, 2.0 ** 15))
    assert all(torch.isfinite(x).all() for n, x in big.items() if n == "dq")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_same_bits_every_time(cuda, dtype):
    args = inputs(14, 4, 200, 200, 8, 2, 64, dtype, cuda, 16, 40)
    a = run(*args[:4], causal=True, bias=args[4], buckets=args[5], drop=26, seed=1)
    for _ in range(3):
        b = run(*args[:4], causal=True, bias=args[4], buckets=args[5], drop=26, seed=1)
        assert all(torch.equal(a[n], b[n]) for n in a)


def test_runs_on_the_current_stream(cuda):
    args = inputs(15, 2, 90, 90, 4, 2, 64, BF16, cuda, 8, 16)
    want = run(*args[:4], bias=args[4], buckets=args[5])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(int(6e8))          # the default stream is busy for about a quarter second
    with torch.cuda.stream(side):
        got = run(*args[:4], bias=args[4], buckets=args[5])
    side.synchronize()
    busy = not torch.cuda.default_stream().query()
    torch.cuda.synchronize()
    assert busy, "an op launched on, or waited for, the default stream"
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_graph_replays_with_new_seeds(cuda):
    q, k, v, g, bias, where = inputs(16, 2, 100, 100, 4, 2, 64, BF16, cuda, 8, 16)
    leaves = [t.requires_grad_() for t in (q, k, v, bias)]
    seed = torch.zeros(1, dtype=torch.int64, device=cuda)

    def step():
        out = d2p_amd.attention(*leaves[:3], causal=True, bias=leaves[3], buckets=where,
                                dropout=0.2, seed=seed)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for n in range(4):
        seed.fill_(1000 + n)
        graph.replay()
        got = [o.clone() for o in outs]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n


def test_autocast_and_second_derivatives(cuda):
    q, k, v, g, bias, where = inputs(17, 1, 40, 40, 2, 2, 32, F32, cuda, 4, 8)
    with torch.autocast("cuda", dtype=BF16):
        out = d2p_amd.attention(q, k, v, bias=bias, buckets=where)
    assert out.dtype == BF16
    assert torch.equal(out, d2p_amd.attention(q.to(BF16), k.to(BF16), v.to(BF16), bias=bias, buckets=where))
    q.requires_grad_()
    dq, = torch.autograd.grad(d2p_amd.attention(q, k, v), q, g, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        dq.sum().backward()


def test_refusals(cuda):
    q, k, v, _, bias, where = inputs(18, 2, 8, 8, 4, 2, 32, F32, cuda, 4, 2)
    f = d2p_amd.attention
    bad = [
        (dict(q=q.double()), "float32, float16 or bfloat16"),
        (dict(q=q[0]), "4D"),
        (dict(k=k.to(BF16)), "q's type"),
        (dict(v=v[:, :7]), "same shape"),
        (dict(q=q[:1]), "batch size"),
        (dict(q=q[..., :16]), "head size"),
        (dict(q=q[..., :12].contiguous(), k=k[..., :12].contiguous(), v=v[..., :12].contiguous()),
         "multiple of 8"),
        (dict(q=q[:, :, :3]), "multiple of key heads"),
        (dict(k=k.cpu()), "CUDA tensor"),
        (dict(lengths=torch.zeros(2, 2, device=cuda)), "lengths must be"),
        (dict(lengths=torch.zeros(3, 2, dtype=torch.int32, device=cuda)), r"\[B, 2\]"),
        (dict(lengths=torch.zeros(2, 2, dtype=torch.int32)), "CUDA tensor"),
        (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
        (dict(bias=bias), "go together"), (dict(buckets=where), "go together"),
        (dict(bias=bias[:, :2], buckets=where), "bias must be"),
        (dict(bias=bias.to(F16), buckets=where), "bias must be"),
        (dict(bias=bias, buckets=where[:4]), "buckets must be"),
        (dict(bias=bias, buckets=where.long()), "buckets must be"),
        (dict(dropout=1.0, seed=1), "dropout"), (dict(dropout=-0.1, seed=1), "dropout"),
        (dict(dropout=0.001, seed=1), "256ths"),
        (dict(dropout=0.5, seed=torch.zeros(1, device=cuda)), "seed must be"),
        (dict(dropout=0.5, seed=torch.zeros(2, dtype=torch.int64, device=cuda)), "one number"),
    ]
    for kw, match in bad:
        a = dict(q=q, k=k, v=v)
        a.update(kw)
        with pytest.raises(RuntimeError, match=match):
            f(**a)
    with pytest.raises(ValueError, match="seed"):
        f(q, k, v, dropout=0.5)


def test_empty_tensors(cuda):
    for B, Lq, Lk in itertools.product((0, 2), (0, 5), (0, 6)):
        args = inputs(19, B, Lq, Lk, 2, 2, 16, BF16, cuda, 4, 2)
        got = run(*args[:4], bias=args[4], buckets=args[5])
        assert got["out"].shape == (B, Lq, 2, 16)
        if B == 0 or Lq == 0 or Lk == 0:
            assert all((x == 0).all() for x in got.values())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("R", [16, 130, 1024])
def test_bias_gradient_beside_blocks_without_keys(cuda, R, causal, dtype):
    """Blocks of queries past nq, of elements without keys and (causal) before the first key add
    nothing to the bias's gradient, whatever the workgroups before them left in LDS."""
    ls = lens(cuda, (520, 140), (3, 140), (100, 0), (0, 0), (520, 1), (0, 140), (130, 7), (520, 0))
    args = inputs(23, len(ls), 520, 140, 2, 1, 64, dtype, cuda, 12, R)
    got = both(args, lengths=ls, causal=causal)
    for _ in range(5):
        again = run(*args[:4], ls, causal, None, *args[4:])
        assert all(torch.equal(got[n], again[n]) for n in got)
    # nothing but such blocks
    ls = lens(cuda, *[(0, 140), (520, 0), (0, 0), (130, 0)] * 2)
    assert all((x == 0).all() for x in run(*args[:4], ls, causal, None, *args[4:]).values())


HALF_SIZES = [(2, 40, 40, 2, 2, 32), (1, 3, 400, 4, 2, 64), (1, 3, 1500, 2, 1, 64), (1, 200, 130, 2, 1, 128)]


@pytest.mark.parametrize("low", [-2e7, -1e8, -1e9, torch.finfo(F32).min])
@pytest.mark.parametrize("size", HALF_SIZES, ids=str)
def test_half_beside_low_biases_in_32_bits(cuda, size, low):
    """Rows whose every bias is the same low number keep probabilities that sum to one in the
    backward pass, from either forward.  So the sum of dv over the keys is that of the gradients:
    P and dv are rounded to half once each, the statistics are good to 2^-18.  Below -2^29 a score
    adds nothing to its bias, and everything is what equal scores give."""
    q, k, v, g, _, where = inputs(21, *size, F16, cuda, 3, 20)
    B, Lq, Lk, Hq, Hkv, D = size
    bias = torch.full((3, Hq), low, device=cuda)
    got = run(q, k, v, g, bias=bias, buckets=where)
    assert all(x.isfinite().all() for x in got.values())
    u = ref.U[F16]
    have = got["dv"].double().sum(1)
    join = lambda x: x.double().sum(1).view(B, Hkv, Hq // Hkv, D).sum(2)  # noqa: E731
    bound = (2 * u + 2.0 ** -18) * join(g.abs()) + Lk * ref.TINY[F16]
    assert ((have - join(g)).abs() <= bound).all()
    if low < -2.0 ** 29:
        tiny = 2.0 ** -40          # a scale that leaves the scores equal in 64 bits, undone
        want, err = ref.attention(q, k, v, g, scale=tiny, bias=bias * 0, buckets=where)
        for n in ("dq", "dk"):
            f = D ** -0.5 / tiny
            want[n], err[n] = want[n] * f, (err[n] - ref.TINY[F16]) * f + ref.TINY[F16]
        check(got, want, err)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_bias_of_distances_that_only_padded_queries_have(cuda, causal, D, dtype):
    """NaN, infinity or a bucket that does not exist, at distances that no pair within the
    lengths has, changes no bit; that bucket's gradient is zero."""
    nq, nk = 40, 60
    q, k, v, g, bias, _ = inputs(22, 1, 100, 60, 2, 1, D, dtype, cuda, 2, 64)
    ls = lens(cuda, (nq, nk))
    lowest = -nq + 1 - (nk - nq if causal else 0)         # the smallest j - at_i within the lengths
    where = torch.tensor([int(d < lowest) for d in range(-64, 65)], dtype=torch.int32, device=cuda)
    if causal:
        # ahead of a query no pair is seen, but padded queries of the same tile see those
        where[64 + 1:] = 1
    bias[1] = 0
    want = run(q, k, v, g, ls, causal, None, bias, where)
    assert (want["dbias"][1] == 0).all()
    gone = where.clone()
    gone[where == 1] = 7
    for value, place in ((float("nan"), where), (float("inf"), where), (0.0, gone)):
        bias[1] = value
        got = run(q, k, v, g, ls, causal, None, bias, place)
        assert all(torch.equal(got[n], want[n]) for n in want), value
