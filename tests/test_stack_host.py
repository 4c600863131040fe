"""The operators around a sequence encoder's attention layers on the host (no GPU needed): the C
ABI's checks of its arguments, fakes, refusal of CPU tensors and tangents, the oracle itself.
"""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import _capi
import _stackref as ref
import d2p_amd

HEADER = os.path.join(_capi.ROOT, "include", "d2p_amd_training.h")
FAKE = ctypes.c_void_p(0x1000)      # non-null, never dereferenced by the host checks
P, I, F, Z, LL = (ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t,
                  ctypes.c_longlong)
NAN, INF = float("nan"), float("inf")


class Strides(ctypes.Structure):
    _fields_ = [("batch", LL), ("row", LL)]


class Vector(ctypes.Structure):
    _fields_ = [("data", P), ("dtype", I)]


class Embedding(ctypes.Structure):
    _fields_ = [("weight_dtype", I), ("dtype", I), ("B", I), ("L", I), ("V", I), ("D", I),
                ("tokens", P), ("token_bytes", I), ("lengths", P), ("padding", LL), ("scale", F),
                ("grad", Strides)]


class Residual(ctypes.Structure):
    _fields_ = [("dtype", I), ("block_dtype", I), ("B", I), ("L", I), ("D", I), ("with_y", I),
                ("x", Strides), ("y", Strides), ("dh", Strides), ("dn", Strides), ("norm", I),
                ("post_norm", I), ("weight", Vector), ("bias", Vector), ("post_weight", Vector),
                ("post_bias", Vector), ("gate_kind", I), ("gate", P), ("gate_dtype", I),
                ("gate_strides", Strides), ("scale", F), ("residual_scale", F), ("eps", F)]


class Tensor(ctypes.Structure):
    _fields_ = [("src", P), ("dst", P), ("n", LL), ("dtype", I)]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_capi.LIB_PATH):
        pytest.skip("libd2p_amd.so not built (run __graft_entry__.build())")
    lib = ctypes.CDLL(_capi.LIB_PATH)
    lib.d2p_last_error.restype = ctypes.c_char_p
    for n, a in (("d2p_token_embedding_backward_workspace_bytes", P),
                 ("d2p_residual_norm_backward_workspace_bytes", P),
                 ("d2p_global_norm_workspace_bytes", I)):
        getattr(lib, n).restype = Z
        getattr(lib, n).argtypes = [a]
    lib.d2p_token_embedding.argtypes = [P] * 4
    lib.d2p_token_embedding_backward.argtypes = [P] * 4 + [Z, P]
    lib.d2p_residual_norm.argtypes = [P] * 7
    lib.d2p_residual_norm_backward.argtypes = [P] * 14 + [Z, P]
    lib.d2p_global_norm.argtypes = [P, I, P, P, Z, P]
    lib.d2p_clip_by_norm.argtypes = [P, I, ctypes.c_double, P, P, Z, P]
    return lib


def said(lib):
    return lib.d2p_last_error().decode()


def embedding(**kw):
    a = dict(weight_dtype=0, dtype=2, B=2, L=8, V=50, D=64, tokens=FAKE, token_bytes=8, padding=-1,
             scale=1.0, grad=Strides(512, 64))
    a.update(kw)
    return Embedding(**a)


def residual(**kw):
    rows = Strides(512, 64)
    a = dict(dtype=0, block_dtype=2, B=2, L=8, D=64, with_y=1, x=rows, y=rows, dh=rows, dn=rows,
             norm=1, scale=1.0, residual_scale=1.0, eps=1e-6)
    a.update(kw)
    return Residual(**a)


def test_every_declared_function_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(d2p_\w+)\s*\(", text)))
    assert len(names) == 9
    out = subprocess.run(["nm", "-D", "--defined-only", _capi.LIB_PATH], capture_output=True,
                         text=True, check=True).stdout
    exported = set(re.findall(r"\s[TW]\s+(d2p_\w+)$", out, flags=re.M))
    assert not [n for n in names if n not in exported]


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "element types"), (dict(weight_dtype=1, dtype=2), "pair"),
    (dict(weight_dtype=2, dtype=0), "pair"), (dict(B=-1), "negative"), (dict(L=-2), "negative"),
    (dict(B=1 << 16, L=1 << 15), "too many"), (dict(V=0), "between 1"),
    (dict(V=2 ** 31 - 1), "between 1"), (dict(D=7), "features"), (dict(D=(1 << 20) + 1), "features"),
    (dict(token_bytes=2), "bytes"), (dict(padding=50), "padding"), (dict(padding=-2), "padding"),
    (dict(scale=NAN), "finite"), (dict(scale=INF), "finite")], ids=str)
def test_embedding_checks(lib, kw, match):
    p = ctypes.byref(embedding(**kw))
    assert lib.d2p_token_embedding(p, FAKE, FAKE, None) == 1 and match in said(lib)
    assert lib.d2p_token_embedding_backward(p, FAKE, FAKE, FAKE, 1 << 40, None) == 1
    assert match in said(lib)


def test_embedding_pointers_and_workspaces(lib):
    p = embedding()
    b = ctypes.byref(p)
    assert lib.d2p_token_embedding(None, FAKE, FAKE, None) == 1
    for args in ((None, FAKE), (FAKE, None)):
        assert lib.d2p_token_embedding(b, *args, None) == 1 and "null" in said(lib)
    need = lib.d2p_token_embedding_backward_workspace_bytes(b)
    assert need >= 16 * 4
    for args in ((None, FAKE), (FAKE, None)):
        assert lib.d2p_token_embedding_backward(b, *args, FAKE, need, None) == 1 and "null" in said(lib)
    assert lib.d2p_token_embedding_backward(b, FAKE, FAKE, FAKE, need - 1, None) == 1
    assert "workspace" in said(lib)
    assert lib.d2p_token_embedding_backward(b, FAKE, FAKE, ctypes.c_void_p(0x1008), need, None) == 1
    assert "aligned" in said(lib)
    bad = embedding(tokens=None)
    assert lib.d2p_token_embedding(ctypes.byref(bad), FAKE, FAKE, None) == 1 and "null" in said(lib)
    empty = embedding(B=0, tokens=None)
    assert lib.d2p_token_embedding(ctypes.byref(empty), None, None, None) == 0
    assert lib.d2p_token_embedding_backward_workspace_bytes(None) == 0
    assert lib.d2p_token_embedding_backward_workspace_bytes(ctypes.byref(embedding(V=0))) == 0
    for B, L, V, D in ((1, 1, 1, 8), (1, 1 << 20, 70000, 512), (1 << 15, 1 << 15, 4, 64),
                       (1, 1, 2 ** 31 - 2, 8), (3, 4099, 4097, 200), (1, 2 ** 31 - 1, 40, 8)):
        big = embedding(B=B, L=L, V=V, D=D)
        assert lib.d2p_token_embedding_backward_workspace_bytes(ctypes.byref(big)) > 0


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=5), "element types"), (dict(dtype=1, block_dtype=2), "pair"), (dict(B=-1), "negative"),
    (dict(B=1 << 20, L=1 << 11), "too many"), (dict(D=7), "features"), (dict(D=8193), "features"),
    (dict(norm=3), "norm"), (dict(post_norm=-1), "norm"), (dict(weight=Vector(0x1000, 7)), "vector"),
    (dict(post_bias=Vector(0x1000, -1)), "vector"), (dict(gate_kind=4), "gate"),
    (dict(norm=0, weight=Vector(0x1000, 0)), "need the norm"),
    (dict(post_bias=Vector(0x1000, 0)), "need the norm"),
    (dict(gate_kind=1, gate=FAKE, gate_dtype=1), "gate must"), (dict(gate_kind=2), "null"),
    (dict(eps=-1.0), "eps"), (dict(eps=NAN), "eps")], ids=str)
def test_residual_checks(lib, kw, match):
    p = ctypes.byref(residual(**kw))
    assert lib.d2p_residual_norm(p, FAKE, FAKE, FAKE, FAKE, FAKE, None) == 1 and match in said(lib)
    assert lib.d2p_residual_norm_backward(p, *[FAKE] * 13, 1 << 40, None) == 1 and match in said(lib)


def test_residual_pointers_and_workspaces(lib):
    p = residual()
    b = ctypes.byref(p)

    def forward(x=FAKE, y=FAKE, h=FAKE, n=FAKE, p=b):
        return lib.d2p_residual_norm(p, x, y, h, n, None, None), said(lib)

    for kw, match in ((dict(x=None), "null"), (dict(n=None), "null"), (dict(y=None), "together"),
                      (dict(h=None), "together"), (dict(y=None, h=None), "together")):
        rc, message = forward(**kw)
        assert rc == 1 and match in message
    first = ctypes.byref(residual(with_y=0, post_norm=1))
    rc, message = forward(y=None, h=None, p=first)
    assert rc == 1 and "needs y" in message
    need = lib.d2p_residual_norm_backward_workspace_bytes(b)

    def backward(dh=FAKE, dn=FAKE, stream=FAKE, y=FAKE, stats=FAKE, dx=FAKE, dy=FAKE, dgate=None,
                 ws=FAKE, bytes=need, p=b):
        return lib.d2p_residual_norm_backward(p, dh, dn, stream, y, stats, dx, dy, dgate, None, None,
                                              None, None, ws, bytes, None), said(lib)

    half = ctypes.byref(residual(dtype=2))
    post = ctypes.byref(residual(post_norm=2))
    for kw, match in ((dict(dh=None, dn=None), "dh or dn"), (dict(dx=None), "null"),
                      (dict(stream=None), "null"), (dict(stats=None), "null"),
                      (dict(y=None, p=half), "y is needed"), (dict(y=None, dgate=FAKE), "y is needed"),
                      (dict(y=None, p=post), "null"), (dict(dy=None), "dy is not dx"),
                      (dict(dy=None, p=post), "dy is not dx"), (dict(p=first), "dy needs y"),
                      (dict(dy=None, p=first), "dy is not dx"),
                      (dict(p=ctypes.byref(residual(with_y=0))), "dy needs y"),
                      (dict(stats=ctypes.c_void_p(0x1004)), "aligned"), (dict(ws=None), "workspace"),
                      (dict(bytes=need - 1), "workspace")):
        rc, message = backward(**kw)
        assert rc == 1 and match in message, (kw, message)
    empty = ctypes.byref(residual(B=0))
    assert lib.d2p_residual_norm(empty, None, None, None, None, None, None) == 0
    assert lib.d2p_residual_norm_backward_workspace_bytes(None) == 0
    for B, L, D, kind in ((1, 1, 8, 0), (1 << 15, 3, 512, 2), (4, 1 << 20, 8192, 1), (3, 0, 64, 2)):
        big = residual(B=B, L=L, D=D, gate_kind=kind, gate=FAKE)
        assert lib.d2p_residual_norm_backward_workspace_bytes(ctypes.byref(big)) > 0


def test_clip_checks(lib):
    def call(tensors, count=None, max_norm=1.0, norm=FAKE, ws=FAKE, bytes=1 << 20):
        list = (Tensor * max(1, len(tensors)))(*tensors)
        n = len(tensors) if count is None else count
        rcs = (lib.d2p_clip_by_norm(list, n, max_norm, norm, ws, bytes, None),
               lib.d2p_global_norm(list, n, norm, ws, bytes, None) if max_norm == 1.0 else 1)
        return rcs, said(lib)

    good = Tensor(0x1000, 0x2000, 10, 0)
    for args, kw, match in (([[good]], dict(norm=None), "null"), ([[good]], dict(count=-1), "null"),
                            ([[good]], dict(ws=None), "workspace"), ([[good]], dict(bytes=100), "workspace"),
                            ([[good]], dict(ws=ctypes.c_void_p(0x1004)), "aligned"),
                            ([[good, Tensor(0x1000, 0x2000, 10, 3)]], {}, "element type"),
                            ([[Tensor(0x1000, 0x2000, -1, 0)]], {}, "negative"),
                            ([[Tensor(0, 0x2000, 1, 0)]], {}, "null"),
                            ([[Tensor(0x1002, 0x2000, 1, 0)]], {}, "aligned"),
                            ([[Tensor(0x1001, 0x2000, 1, 2)]], {}, "aligned"),
                            ([[Tensor(0x1000, 0x2000, 1 << 42, 2)]], {}, "too long")):
        rcs, message = call(*args, **kw)
        assert rcs == (1, 1) and match in message, (kw, message)
    for bad in (-1.0, NAN):
        rcs, message = call([good], max_norm=bad)
        assert rcs[0] == 1 and "max_norm" in message
    rcs, _ = call([Tensor(0x1000, 0, 1, 0)], max_norm=2.0)      # no place for the result
    assert rcs[0] == 1
    assert lib.d2p_global_norm_workspace_bytes(0) >= 8 * 1024
    assert lib.d2p_global_norm_workspace_bytes(1000) - lib.d2p_global_norm_workspace_bytes(0) == 22000


def test_cpu_tensors_fail_loudly():
    x, t = torch.randn(1, 4, 16), torch.zeros(1, 4, dtype=torch.int64)
    w = torch.randn(5, 16, requires_grad=True)
    for call in (lambda: d2p_amd.token_embedding(t, w), lambda: d2p_amd.residual_norm(x, x),
                 lambda: d2p_amd.residual_norm(x), lambda: d2p_amd.global_norm([x]),
                 lambda: d2p_amd.clip_gradients([x], 1.0),
                 lambda: d2p_amd.clip_gradients([x], 1.0, out=[x]),
                 lambda: d2p_amd.SequenceEncoder(5, 16, 2, 1)(t)):
        with pytest.raises(RuntimeError, match="HIP"):
            call()


def test_python_layer_checks():
    x, t, w = torch.zeros(1, 4, 16), torch.zeros(1, 4, dtype=torch.int64), torch.zeros(5, 16)
    v = torch.ones(16)
    op = d2p_amd.residual_norm
    for call, match in ((lambda: op(x, x, norm="mean"), "norm must"),
                        (lambda: op(x, x, post_norm="none"), "post_norm must"),
                        (lambda: op(x, post_norm="rms"), "need y"), (lambda: op(x, gate=v), "need y"),
                        (lambda: op(x, residual_scale=2.0), "need y"),
                        (lambda: op(x, norm=None), "nothing to do"),
                        (lambda: op(x, x, v, norm=None), "need norm"),
                        (lambda: op(x, x, post_bias=v), "need post_norm"),
                        (lambda: op(x, x, dtype=torch.half), "dtype is y's"),
                        (lambda: d2p_amd.token_embedding(t, w, padding=5), "padding"),
                        (lambda: d2p_amd.clip_gradients([], 1.0), "at least one"),
                        (lambda: d2p_amd.clip_gradients([x], 1.0, out=[x, x]), "1 tensors"),
                        (lambda: d2p_amd.SequenceEncoder(5, 16, 2, 1, norm=None), "norm"),
                        (lambda: d2p_amd.SequenceEncoder(5, 16, 2, 1, post_norm="l"), "post_norm"),
                        (lambda: d2p_amd.SequenceEncoder(5, 16, 2, 1, padding=5), "padding")):
        with pytest.raises(ValueError, match=match):
            call()
    assert float(d2p_amd.clip_grad_norm_([v], 1.0)) == 0.0        # no gradient at all


def test_clipping_nothing_gives_zero_where_the_parameters_are():
    for device in ("cpu", "meta"):
        p = torch.nn.Parameter(torch.zeros(3, device=device))
        norm = d2p_amd.clip_grad_norm_(iter([p]), 1.0)
        assert norm.device == p.device and norm.shape == () and norm.dtype == torch.float32
    assert float(d2p_amd.clip_grad_norm_([], 1.0)) == 0.0


def test_encoder_parameters():
    m = d2p_amd.SequenceEncoder(21, 32, 4, 3, 2, norm="layer", post_norm="layer", gated=0.1,
                                num_buckets=8, padding=20, scale=2.0)
    shapes = {k: tuple(v.shape) for k, v in m.named_parameters()}
    assert shapes["embedding"] == (21, 32) and len(m.layers) == 3
    for name, n in (("weights", 4), ("biases", 4), ("post_weights", 3), ("post_biases", 3), ("gates", 3)):
        assert [shapes[f"{name}.{i}"] for i in range(n)] == [(32,)] * n and f"{name}.{n}" not in shapes
    assert m.gates[0][0].item() == pytest.approx(0.1) and (m.weights[0] == 1.0).all()
    assert m.layers[0].qkv.weight.shape == ((4 + 2 * 2) * 8, 32) and m.layers[2].bias.shape == (8, 4)
    plain = d2p_amd.SequenceEncoder(21, 32, 4, 0)
    assert sorted(dict(plain.named_parameters())) == ["embedding", "weights.0"]


def test_fakes_give_output_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    o = torch.ops.d2p_amd
    with FakeTensorMode():
        t = torch.zeros(2, 5, dtype=torch.int64, device="cuda")
        w = torch.empty(7, 16, device="cuda")
        out = d2p_amd.token_embedding(t, w, dtype=torch.half)
        assert out.shape == (2, 5, 16) and out.dtype == torch.half
        dw = o.token_embedding_backward(out, t, None, 1.0, -1, 7, torch.float32)
        assert dw.shape == (7, 16) and dw.dtype == torch.float32
        x, y = torch.empty(2, 5, 16, device="cuda"), torch.empty(2, 5, 16, device="cuda", dtype=torch.half)
        h, n = d2p_amd.residual_norm(x, y)
        assert h.shape == n.shape == x.shape and (h.dtype, n.dtype) == (torch.float32, torch.half)
        h, n = d2p_amd.residual_norm(x, dtype=torch.half)
        assert h is x and n.dtype == torch.half
        v = torch.empty(16, device="cuda")
        h, n, st = o.residual_norm_forward(x, y, v, None, None, None, v, 1, 0, 1.0, 1.0, 1e-6, torch.half, True)
        assert st.shape == (2, 5, 4) and st.dtype == torch.float32
        g = o.residual_norm_backward(x, y, h, y, st, v, None, None, None, v, 1, 0, 1.0, 1.0, 1e-6,
                                     torch.half, True, 3)
        assert [None if t is None else tuple(t.shape) for t in g] == \
            [(2, 5, 16), (2, 5, 16), (16,), (16,), None, None, None]
        out, norm = d2p_amd.clip_gradients([x, y], 1.0)
        assert [t.dtype for t in out] == [torch.float32, torch.half] and norm.shape == ()
        assert d2p_amd.global_norm([x, y]).dtype == torch.float32


def test_forward_mode_raises():
    """No operator has a derivative in forward mode: a tangent raises, on whichever input, and is
    never dropped (meta tensors: the operators' autograd layer without their kernels)."""
    import torch.autograd.forward_ad as fwd
    m = dict(device="meta")
    t, w = torch.zeros(2, 5, dtype=torch.int64, **m), torch.empty(7, 16, **m)
    x, v = torch.empty(2, 5, 16, **m), torch.empty(16, **m)

    def norm(x, y, a, b, c, d, g):
        return d2p_amd.residual_norm(x, y, a, b, norm="layer", post_norm="layer", post_weight=c,
                                     post_bias=d, gate=g)

    for f, args in ((lambda w: d2p_amd.token_embedding(t, w), (w,)), (norm, (x, x, v, v, v, v, v)),
                    (lambda x: d2p_amd.residual_norm(x)[1], (x,)),
                    (lambda x: d2p_amd.global_norm([x, v]), (x,)),
                    (lambda x: d2p_amd.clip_gradients([v, x], 1.0)[0][1], (x,))):
        f(*args)
        for n, a in enumerate(args):
            def of(b):
                return f(*args[:n], b, *args[n + 1:])
            with pytest.raises(RuntimeError, match="forward AD"):
                torch.func.jvp(of, (a,), (torch.ones_like(a),))
            with torch.no_grad(), fwd.dual_level(), pytest.raises(RuntimeError, match="forward AD"):
                of(fwd.make_dual(a, torch.ones_like(a)))
    for f, a in ((lambda a: d2p_amd.token_embedding(t, a), w), (lambda a: d2p_amd.residual_norm(a, x)[0], x)):
        a = a.detach().requires_grad_()
        out = f(a)
        g = torch.ones_like(out)
        torch.autograd.grad(out, a, g, retain_graph=True)
        with fwd.dual_level(), pytest.raises(RuntimeError, match="forward AD"):
            torch.autograd.grad(out, a, fwd.make_dual(g, g))


# ------------------------------------------------------------------ the oracle's own parts

FORMS = [("rms", None, None), ("layer", "rms", "feature"), ("rms", "layer", "sequence"),
         ("layer", "layer", "token"), (None, "layer", "token"), (None, None, "feature")]


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_oracle_gradient_against_differences(form):
    """The 64-bit residual norm the kernels are checked with, against its own differences: with
    h = 1e-5 the truncation h^2 f''' / 6 and the rounding 1e-16 f / h are both below 1e-8."""
    norm, post, gate = form
    g = torch.Generator().manual_seed(1)
    B, L, D = 2, 3, 10

    def randn(*s):
        return torch.randn(s, generator=g, dtype=torch.float64)

    s = dict(x=randn(B, L, D), y=randn(B, L, D))
    if gate:
        s["gate"] = randn(*{"feature": (D,), "sequence": (B, 1, D), "token": (B, L, D)}[gate])
    for name, kind in (("", norm), ("post_", post)):
        if kind:
            s[name + "weight"], s[name + "bias"] = randn(D), randn(D)
    dh, dn = randn(B, L, D), randn(B, L, D)
    kw = dict(norm=norm, post_norm=post, scale=0.7, residual_scale=1.3, eps=1e-3)
    res, _ = ref.residual(**s, dh=dh, dn=dn, **kw)
    for name in s:
        d = randn(*s[name].shape)

        def f(t):
            r, _ = ref.residual(**{**s, name: s[name] + t * d}, **kw)
            return (r["h"] * dh).sum() + ((r["n"] * dn).sum() if norm else 0.0)

        assert abs((f(1e-5) - f(-1e-5)) / 2e-5 - (res["d" + name] * d).sum()) < 1e-7, name


def test_oracle_against_torch():
    g = torch.Generator().manual_seed(2)
    t = torch.randint(0, 9, (3, 7), generator=g)
    w = torch.randn(9, 8, generator=g, dtype=torch.float64, requires_grad=True)
    grad = torch.randn(3, 7, 8, generator=g, dtype=torch.float64)
    out, _, dw, _ = ref.embedding(t, w, scale=2.0, padding=4, grad=grad)
    want = 2.0 * torch.nn.functional.embedding(t, w) * (t != 4)[..., None]
    assert (out - want).abs().max() < 1e-14
    assert (dw - torch.autograd.grad(want, w, grad)[0]).abs().max() < 1e-13
    out, _, dw, _ = ref.embedding(t, w, torch.tensor([7, 0, 3]), grad=grad)
    assert not out[1].any() and not out[2, 3:].any() and torch.equal(out[0], w[t[0]].detach())
    x = torch.randn(2, 3, 8, generator=g, dtype=torch.float64)
    a, b = torch.randn(8, generator=g).double(), torch.randn(8, generator=g).double()
    r, _ = ref.residual(x, None, a, b, norm="layer", eps=1e-5)
    assert (r["n"] - torch.nn.functional.layer_norm(x, (8,), a, b, 1e-5)).abs().max() < 1e-13
    r, _ = ref.residual(x, None, a, norm="rms", eps=1e-5)
    assert (r["n"] - torch.nn.functional.rms_norm(x, (8,), a, 1e-5)).abs().max() < 1e-13
