"""residual_norm and its gradients against the formulas in 64 bits (tests/_stackref.py)."""
import pytest
import torch

import _stackref as ref
import d2p_amd

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAMES = ("x", "y", "gate", "weight", "bias", "post_weight", "post_bias")


def inputs(B, L, D, dtype, block, norm="rms", post=None, gate=None, first=False, vectors=F32,
           seed=0, gate_type=None, offset=0.0):
    g = torch.Generator().manual_seed(seed)

    def randn(*shape, to, scale=1.0, mean=0.0):
        return (mean + scale * torch.randn(shape, generator=g)).to(to)

    s = dict.fromkeys(NAMES)
    s["x"] = randn(B, L, D, to=dtype, scale=2.0, mean=offset)
    if not first:
        s["y"] = randn(B, L, D, to=block, mean=offset)
    shape = {"feature": (D,), "sequence": (B, 1, D), "token": (B, L, D)}.get(gate)
    if shape:
        s["gate"] = randn(*shape, to=gate_type or (F32 if gate == "feature" else block))
    for name, kind in (("", norm), ("post_", post)):
        if kind:
            s[name + "weight"] = randn(D, to=vectors, scale=0.3, mean=1.0)
        if kind == "layer":
            s[name + "bias"] = randn(D, to=vectors)
    grads = randn(B, L, D, to=dtype), randn(B, L, D, to=block)
    return s, grads


def run(s, dh, dn, dev="cuda", **kw):
    leaves = {k: v.to(dev).requires_grad_() for k, v in s.items() if v is not None}
    h, n = d2p_amd.residual_norm(leaves["x"], leaves.get("y"), leaves.get("weight"),
                                 leaves.get("bias"), post_weight=leaves.get("post_weight"),
                                 post_bias=leaves.get("post_bias"), gate=leaves.get("gate"), **kw)
    got = {}
    if "y" in leaves:
        got["h"] = h
    if n is not None:
        got["n"] = n
    outs = [(h, dh)] if dh is not None else []
    outs += [(n, dn)] if dn is not None and n is not None else []
    if outs:
        grads = torch.autograd.grad([o for o, _ in outs], list(leaves.values()),
                                    [g.to(dev) for _, g in outs], allow_unused=True)
        got.update({"d" + k: g for k, g in zip(leaves, grads) if g is not None})
    return got


def check(s, dh, dn, **kw):
    got = run(s, dh, dn, **kw)
    want, off = ref.residual(**s, dh=dh, dn=dn, **kw)
    if s["y"] is None and dh is not None:       # h is x: its gradient joins by itself
        raise AssertionError("not a case of this function")
    for name, value in want.items():
        a = got[name].detach().cpu().double()
        assert a.shape == value.shape, name
        err = (a - value).abs()
        assert (err <= off[name]).all(), (name, float((err - off[name]).max()), float(err.max()))
    for name in got:
        source = s.get(name[1:]) if name.startswith("d") else None
        if source is not None:
            assert got[name].dtype == source.dtype and got[name].shape == source.shape
    again = run(s, dh, dn, **kw)
    assert all(torch.equal(got[k], again[k]) for k in got)
    return got


PAIRS = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)]
SIZES = [(1, 1, 8), (3, 5, 15), (2, 9, 9), (2, 33, 64), (3, 17, 96), (2, 11, 200), (5, 23, 333),
         (2, 40, 512), (2, 7, 520), (3, 5, 1000), (2, 6, 2048), (1, 5, 2055), (1, 3, 4100),
         (2, 2, 8192), (1, 700, 24), (70, 3, 32)]
FORMS = [  # norm, post_norm, gate, scale, residual_scale
    ("rms", None, None, 1.0, 1.0),
    ("rms", "rms", "feature", 1.0, 1.0),
    ("layer", "layer", "token", 0.5, 1.25),
    ("layer", None, "sequence", 0.7, 1.0),
    (None, "layer", "sequence", 1.0, 2.0),
    ("rms", "layer", None, -1.5, 0.5),
    (None, "rms", "feature", 1.0, 1.0),
    (None, None, "token", 1.0, 1.0),
    ("layer", None, None, 2.0, 2.0),
]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(cuda, size):
    B, L, D = size
    for n, (dtype, block) in enumerate(PAIRS):
        for m in (n, n + 4):
            norm, post, gate, scale, rscale = FORMS[(m + B + D) % len(FORMS)]
            s, (dh, dn) = inputs(B, L, D, dtype, block, norm, post, gate, seed=n)
            check(s, dh, dn, norm=norm, post_norm=post, scale=scale, residual_scale=rscale)


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids=str)
def test_forms(cuda, form, pair):
    norm, post, gate, scale, rscale = form
    for B, L, D in ((3, 70, 48), (2, 5, 1032)):
        s, (dh, dn) = inputs(B, L, D, *pair, norm, post, gate)
        kw = dict(norm=norm, post_norm=post, scale=scale, residual_scale=rscale)
        check(s, dh, dn, **kw)
        check(s, dh, None, **kw)            # one result's gradient alone
        if norm:
            check(s, None, dn, **kw)
        check(s, None, None, **kw)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("pair", PAIRS, ids=str)
def test_before_the_first_block(cuda, norm, pair):
    for B, L, D in ((3, 37, 96), (1, 1, 11), (2, 3, 1500)):
        s, (dh, dn) = inputs(B, L, D, *pair, norm, first=True)
        got = check(s, None, dn, norm=norm, dtype=pair[1])
        # h is x, and its gradient joins
        x = s["x"].to(cuda).requires_grad_()
        h, n = d2p_amd.residual_norm(x, None, s["weight"].to(cuda),
                                     None if norm == "rms" else s["bias"].to(cuda), norm=norm,
                                     dtype=pair[1])
        assert h is x
        dx, = torch.autograd.grad((h, n), x, (dh.to(cuda), dn.to(cuda)))
        assert torch.equal(dx, got["dx"] + dh.to(cuda))


@pytest.mark.parametrize("vectors", [F32, F16, BF16])
def test_types_of_vectors_and_gates(cuda, vectors):
    for dtype, block in PAIRS:
        for gate in ("feature", "sequence", "token"):
            for gate_type in {F32, block}:
                s, (dh, dn) = inputs(2, 9, 40, dtype, block, "layer", "layer", gate,
                                     vectors=vectors, gate_type=gate_type)
                check(s, dh, dn, norm="layer", post_norm="layer")


def test_without_vectors(cuda):
    for norm, post in (("rms", "layer"), ("layer", "rms")):
        s, (dh, dn) = inputs(2, 9, 40, F32, F32, norm, post)
        for k in ("weight", "bias", "post_weight", "post_bias"):
            s[k] = None
        check(s, dh, dn, norm=norm, post_norm=post)
    s, (dh, dn) = inputs(2, 9, 40, F32, BF16, "layer", "layer")
    s["weight"] = s["post_weight"] = None       # biases alone
    check(s, dh, dn, norm="layer", post_norm="layer")


def test_values_far_from_zero(cuda):
    """The spread around a mean that is 50 times as large: taken in two passes."""
    s, (dh, dn) = inputs(2, 9, 300, F32, F32, "layer", "layer", "token", offset=100.0)
    check(s, dh, dn, norm="layer", post_norm="layer")
    for D in (40, 700):
        x = torch.full((1, 3, D), 7.25)         # no spread at all
        got = run(dict.fromkeys(NAMES) | dict(x=x), None, torch.ones(1, 3, D), norm="layer", eps=1e-5)
        assert not got["n"].any() and not got["dx"].any()
        zero = run(dict.fromkeys(NAMES) | dict(x=0 * x), None, torch.ones(1, 3, D), eps=1e-4)
        assert not zero["n"].any() and torch.allclose(zero["dx"].cpu(), torch.full_like(x, 100.0))


def test_rows_do_not_touch_each_other(cuda):
    """NaN and infinities stay in their rows (and in sums over rows)."""
    s, (dh, dn) = inputs(2, 9, 72, F32, BF16, "rms", "layer", "token")
    want = run(s, dh, dn, post_norm="layer")
    bad = {k: v if v is None else v.clone() for k, v in s.items()}
    bad["x"][0, 3, 5], bad["y"][1, 2, 7] = float("nan"), float("inf")
    got = run(bad, dh, dn, post_norm="layer")
    rest = torch.ones(2, 9, dtype=torch.bool)
    rest[0, 3] = rest[1, 2] = False
    for k in ("h", "n", "dx", "dy", "dgate"):
        assert torch.equal(got[k].cpu()[rest], want[k].cpu()[rest])
    assert got["n"][0, 3].isnan().all() and got["h"][1, 2].isnan().all()


def test_strides(cuda):
    s, (dh, dn) = inputs(3, 20, 56, BF16, BF16, "layer", "rms", "token")
    kw = dict(norm="layer", post_norm="rms")
    want = run(s, dh, dn, **kw)
    makes = (lambda t: torch.cat((t, t), -1)[..., 56:], lambda t: torch.cat((t, t), 1)[:, 20:],
             lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
             lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
             lambda t: torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape))
    for n, make in enumerate(makes):
        other = makes[(n + 1) % len(makes)]
        t = {k: v if v is None or v.dim() != 3 else (make if k != "y" else other)(v.cuda())
             for k, v in s.items()}
        leaves = {k: v.cuda().detach().requires_grad_() for k, v in t.items() if v is not None}
        h, m = d2p_amd.residual_norm(leaves["x"], leaves["y"], leaves["weight"], leaves["bias"],
                                     post_weight=leaves["post_weight"], gate=leaves["gate"], **kw)
        grads = torch.autograd.grad((h, m), list(leaves.values()), (make(dh.cuda()), other(dn.cuda())))
        got = dict(h=h, n=m) | {"d" + k: g for k, g in zip(leaves, grads)}
        for k in got:
            assert torch.equal(got[k], want[k]), (n, k)
    # broadcast gradients and a broadcast stream
    one = {k: v for k, v in s.items()}
    one["x"] = s["x"][:1, :1].expand(3, 20, 56)
    a = run(one, dh[:, :1].expand_as(dh), dn[:1].expand_as(dn), **kw)
    one["x"] = one["x"].contiguous()
    b = run(one, dh[:, :1].expand_as(dh).contiguous(), dn[:1].expand_as(dn).contiguous(), **kw)
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_empty(cuda):
    for B, L in ((0, 5), (3, 0)):
        s, (dh, dn) = inputs(B, L, 40, F32, BF16, "layer", "layer", "sequence")
        got = run(s, dh, dn, norm="layer", post_norm="layer")
        assert got["h"].shape == (B, L, 40) and got["dgate"].shape == (B, 1, 40)
        for k in ("dgate", "dweight", "dbias", "dpost_weight", "dpost_bias"):
            assert not got[k].any()


def test_some_gradients_only(cuda):
    s, (dh, dn) = inputs(2, 30, 64, BF16, BF16, "layer", "layer", "feature")
    want = run(s, dh, dn, norm="layer", post_norm="layer")
    for keep in (("x",), ("y",), ("weight",), ("post_bias", "gate"), ("bias", "post_weight")):
        t = {k: v.to(cuda) for k, v in s.items()}
        leaves = [t[k].requires_grad_() for k in keep]
        h, n = d2p_amd.residual_norm(t["x"], t["y"], t["weight"], t["bias"], norm="layer",
                                     post_norm="layer", post_weight=t["post_weight"],
                                     post_bias=t["post_bias"], gate=t["gate"])
        got = torch.autograd.grad((h, n), leaves, (dh.to(cuda), dn.to(cuda)))
        assert all(torch.equal(g, want["d" + k]) for g, k in zip(got, keep))


def test_equal_gradients_of_leaves_do_not_share_memory(cuda):
    """x and y have one gradient where nothing stands between them; as leaves they keep one each."""
    x, y = (torch.randn(2, 5, 32, device=cuda, requires_grad=True) for _ in range(2))
    h, n = d2p_amd.residual_norm(x, y)
    (h.square().sum() + n.sum()).backward()
    assert torch.equal(x.grad, y.grad) and x.grad.data_ptr() != y.grad.data_ptr()


def test_refusals(cuda):
    x = torch.zeros(2, 3, 16, device=cuda)
    op = d2p_amd.residual_norm
    for call, match in (
            (lambda: op(x[0], x[0]), "3D"), (lambda: op(x, x[:, :2]), "shape"),
            (lambda: op(x.double(), x.double()), "float32, float16"),
            (lambda: op(x.half(), x), "type"), (lambda: op(x.half(), x.bfloat16()), "type"),
            (lambda: op(x, x, x[0, 0, :8]), "weight must be"), (lambda: op(x, x, gate=x[:, :, :8]), "gate must"),
            (lambda: op(x, x, gate=x[:1]), "gate must"), (lambda: op(x, x, gate=x[:, :2]), "gate must"),
            (lambda: op(x, x.half(), gate=x.bfloat16()), "gate must"),
            (lambda: op(x, x, eps=-1.0), "eps"), (lambda: op(x, x, scale=float("nan")), "finite"),
            (lambda: op(torch.zeros(1, 1, 8200, device=cuda)), "8192"), (lambda: op(x, x.cpu()), "CUDA"),
            (lambda: op(x[..., :7], x[..., :7]), "features")):
        with pytest.raises(RuntimeError, match=match):
            call()


def test_second_derivative_raises(cuda):
    x, y = (torch.randn(2, 5, 32, device=cuda, requires_grad=True) for _ in range(2))
    h, n = d2p_amd.residual_norm(x, y)
    d, = torch.autograd.grad(n.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        d.sum().backward()
