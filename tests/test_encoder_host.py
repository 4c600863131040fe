"""The sequence-encoder operators on the host (no GPU needed): the C ABI's checks of its
arguments, fakes, refusal of CPU tensors, buckets and tables, the oracle's own parts.
"""
import ctypes
import math
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import _capi
import _encoderref as ref
import d2p_amd

HEADER = os.path.join(_capi.ROOT, "include", "d2p_amd_encoder.h")
FAKE = ctypes.c_void_p(0x1000)      # non-null, never dereferenced by the host checks
P, I, F, Z, LL = (ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t,
                  ctypes.c_longlong)


class Strides(ctypes.Structure):
    _fields_ = [("batch", LL), ("row", LL), ("head", LL)]


class Attention(ctypes.Structure):
    _fields_ = [("dtype", I), ("B", I), ("Lq", I), ("Lk", I), ("Hq", I), ("Hkv", I), ("D", I),
                ("q", Strides), ("k", Strides), ("v", Strides), ("grad", Strides), ("lengths", P),
                ("causal", I), ("scale", F), ("bias", P), ("bias_dtype", I), ("num_buckets", I),
                ("buckets", P), ("max_distance", I), ("drop", I), ("seed", ctypes.c_ulonglong),
                ("seed_ptr", P)]


class Norm(ctypes.Structure):
    _fields_ = [("dtype", I), ("B", I), ("L", I), ("Hq", I), ("Hkv", I), ("D", I), ("R", I),
                ("q", Strides), ("k", Strides), ("gq", Strides), ("gk", Strides),
                ("q_weight", P), ("k_weight", P), ("cos", P), ("sin", P), ("table_rows", LL),
                ("positions", P), ("eps", F), ("interleaved", I)]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_capi.LIB_PATH):
        pytest.skip("libd2p_amd.so not built (run __graft_entry__.build())")
    lib = ctypes.CDLL(_capi.LIB_PATH)
    lib.d2p_last_error.restype = ctypes.c_char_p
    for n in ("d2p_attention_workspace_bytes", "d2p_attention_backward_workspace_bytes",
              "d2p_qk_norm_rope_backward_workspace_bytes"):
        getattr(lib, n).restype = Z
        getattr(lib, n).argtypes = [P]
    lib.d2p_attention_forward.argtypes = [P] * 7 + [Z, P]
    lib.d2p_attention_backward.argtypes = [P] * 12 + [Z, P]
    lib.d2p_qk_norm_rope.argtypes = [P] * 6
    lib.d2p_qk_norm_rope_backward.argtypes = [P] * 10 + [Z, P]
    return lib


def attention(**kw):
    rows = Strides(4 * 8 * 64, 4 * 64, 64)
    a = dict(dtype=2, B=2, Lq=8, Lk=8, Hq=4, Hkv=4, D=64, q=rows, k=rows, v=rows, grad=rows,
             scale=0.125)
    a.update(kw)
    return Attention(**a)


def norm(**kw):
    rows = Strides(4 * 8 * 64, 4 * 64, 64)
    a = dict(dtype=2, B=2, L=8, Hq=4, Hkv=4, D=64, R=64, q=rows, k=rows, gq=rows, gk=rows,
             cos=FAKE, sin=FAKE, table_rows=8, eps=1e-6)
    a.update(kw)
    return Norm(**a)


def test_every_declared_function_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(d2p_\w+)\s*\(", text)))
    assert len(names) == 7
    out = subprocess.run(["nm", "-D", "--defined-only", _capi.LIB_PATH], capture_output=True,
                         text=True, check=True).stdout
    exported = set(re.findall(r"\s[TW]\s+(d2p_\w+)$", out, flags=re.M))
    assert not [n for n in names if n not in exported]


BAD_ATTENTION = [
    (dict(dtype=3), "element type"), (dict(B=-1), "negative"), (dict(Lk=-1), "negative"),
    (dict(Hq=4, Hkv=3), "multiple of key heads"), (dict(Hkv=0), "multiple of key heads"),
    (dict(D=60), "head size"), (dict(D=136), "head size"), (dict(D=0), "head size"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(drop=256), "drop"), (dict(drop=-1), "drop"),
    (dict(bias=FAKE, bias_dtype=1, buckets=FAKE, num_buckets=4), "bias must"),
    (dict(bias=FAKE, num_buckets=4), "buckets"), (dict(bias=FAKE, buckets=FAKE), "buckets"),
    (dict(bias=FAKE, buckets=FAKE, num_buckets=4, max_distance=1025), "max_distance"),
    (dict(q=Strides(2048, 260, 64)), "q: strides must be multiples"),
    (dict(k=Strides(2048, 32, 64)), "k: strides must not"),
    (dict(v=Strides(-2048, 256, 64)), "v: strides must not"),
    (dict(k=Strides(2048, 1 << 23, 64)), "k: 128 rows"),
    (dict(Lq=2 ** 31 - 1), "too long"),
    (dict(B=2 ** 30), "too many heads"),
]


@pytest.mark.parametrize("kw,match", BAD_ATTENTION, ids=str)
def test_attention_checks(lib, kw, match):
    p = attention(**kw)
    assert lib.d2p_attention_forward(ctypes.byref(p), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40,
                                     None) == 1
    assert match in lib.d2p_last_error().decode()
    assert lib.d2p_attention_backward(ctypes.byref(p), *[FAKE] * 11, 1 << 40, None) == 1
    assert match in lib.d2p_last_error().decode()


def test_attention_pointers_and_workspaces(lib):
    p = attention()
    b = ctypes.byref(p)
    assert lib.d2p_attention_forward(None, *[FAKE] * 6, 0, None) == 1
    assert lib.d2p_attention_forward(b, None, *[FAKE] * 5, 0, None) == 1
    assert "null" in lib.d2p_last_error().decode()
    assert lib.d2p_attention_forward(b, ctypes.c_void_p(0x1008), *[FAKE] * 5, 0, None) == 1
    assert "aligned" in lib.d2p_last_error().decode()
    need = lib.d2p_attention_backward_workspace_bytes(b)
    assert need >= 2 * 4 * 8 * 4
    assert lib.d2p_attention_backward(b, *[FAKE] * 9, None, FAKE, need - 1, None) == 1
    assert "workspace" in lib.d2p_last_error().decode()
    assert lib.d2p_attention_backward(b, *[FAKE] * 9, FAKE, FAKE, need, None) == 1
    assert "needs a bias" in lib.d2p_last_error().decode()
    bad = attention(grad=Strides(2048, 260, 64))
    assert lib.d2p_attention_backward(ctypes.byref(bad), *[FAKE] * 9, None, FAKE, need, None) == 1
    assert "grad: strides" in lib.d2p_last_error().decode()
    assert lib.d2p_attention_backward_workspace_bytes(None) == 0
    empty = attention(B=0)
    assert lib.d2p_attention_forward(ctypes.byref(empty), *[None] * 6, 0, None) == 0
    assert lib.d2p_attention_backward(ctypes.byref(empty), *[None] * 11, 0, None) == 0


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=-1), "element type"), (dict(L=-1), "negative"), (dict(Hkv=-2), "negative"),
    (dict(D=68), "head size"), (dict(R=65), "even"), (dict(R=130), "even"),
    (dict(R=-2), "even"), (dict(cos=None), "null"), (dict(table_rows=7), "a row for each"),
    (dict(eps=-1.0), "eps")], ids=str)
def test_norm_checks(lib, kw, match):
    p = norm(**kw)
    assert lib.d2p_qk_norm_rope(ctypes.byref(p), FAKE, FAKE, FAKE, FAKE, None) == 1
    assert match in lib.d2p_last_error().decode()
    assert lib.d2p_qk_norm_rope_backward(ctypes.byref(p), *[FAKE] * 9, 1 << 40, None) == 1
    assert match in lib.d2p_last_error().decode()


def test_norm_pointers_and_workspaces(lib):
    p = norm()
    b = ctypes.byref(p)
    assert lib.d2p_qk_norm_rope(b, None, FAKE, FAKE, FAKE, None) == 1
    assert lib.d2p_qk_norm_rope_backward(b, *[FAKE] * 9, 16, None) == 1
    assert "workspace" in lib.d2p_last_error().decode()
    empty = norm(B=0)
    assert lib.d2p_qk_norm_rope(ctypes.byref(empty), None, None, None, None, None) == 0
    assert lib.d2p_qk_norm_rope_backward(ctypes.byref(empty), *[None] * 9, 0, None) == 0


def test_cpu_tensors_fail_loudly():
    x = torch.randn(1, 4, 2, 16)
    for call in (lambda: d2p_amd.attention(x, x, x), lambda: d2p_amd.qk_norm_rope(x, x),
                 lambda: d2p_amd.SequenceAttention(32, 2)(torch.randn(1, 4, 32))):
        with pytest.raises(RuntimeError, match="HIP"):
            call()


def test_fakes_give_output_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q = torch.empty(2, 5, 4, 16, device="cuda", dtype=torch.bfloat16)
        k = torch.empty(2, 7, 2, 16, device="cuda", dtype=torch.bfloat16)
        out = d2p_amd.attention(q, k, k, causal=True)
        assert out.shape == q.shape and out.dtype == q.dtype
        a = (None, True, 0.25, None, None, 0.0, 0, None)
        out, stats = torch.ops.d2p_amd.attention_forward(q, k, k, *a)
        assert stats.shape == (2, 2, 4, 5) and stats.dtype == torch.float32
        g = torch.ops.d2p_amd.attention_backward(q, q, k, k, out, stats, *a, False)
        assert [tuple(t.shape) for t in g[:3]] == [(2, 5, 4, 16), (2, 7, 2, 16), (2, 7, 2, 16)]
        oq, ok = d2p_amd.qk_norm_rope(q, q[:, :, :2])
        assert oq.shape == q.shape and ok.shape == (2, 5, 2, 16)


def test_relative_buckets():
    for n, most, both in ((32, 128, True), (32, 128, False), (16, 40, True), (33, 100, True),
                          (8, 3, True), (1, 5, False), (2, 9, True), (64, 1024, False)):
        got = d2p_amd.relative_buckets(n, most, both)
        assert got.dtype == torch.int32 and got.shape == (2 * most + 1,)
        m = n // 2 if both else n
        exact = m // 2
        for d, b in zip(range(-most, most + 1), got.tolist()):
            assert 0 <= b < n
            if both:
                assert (b >= m) == (d > 0) or m == 0
            elif d > 0:
                assert b == 0
                continue
            a, b = abs(d), b - (m if both and d > 0 else 0)
            if a < exact or a == 0:
                assert b == min(a, m - 1)
            elif 0 < exact < most:
                x = exact + math.log(a / exact) / math.log(most / exact) * (m - exact)
                assert b == min(m - 1, math.floor(x + 1e-9)) or abs(x - round(x)) < 1e-9
        row = got[most:].tolist()
        assert row[1:] == sorted(row[1:])
    for bad in ((1, 10, True), (4, 0, True), (4, 1025, True)):
        with pytest.raises(ValueError):
            d2p_amd.relative_buckets(*bad)


def test_rope_tables():
    cos, sin = d2p_amd.rope_tables(50, 6, base=100.0)
    assert cos.shape == sin.shape == (50, 3) and cos.dtype == torch.float32
    want = 7 * 100.0 ** (-4 / 6)
    assert abs(cos[7, 2] - math.cos(want)) < 1e-7 and abs(sin[7, 2] - math.sin(want)) < 1e-7
    with pytest.raises(ValueError):
        d2p_amd.rope_tables(4, 5)


def test_python_layer_checks():
    x = torch.randn(1, 4, 2, 16)
    with pytest.raises(ValueError, match="seed"):
        d2p_amd.attention(x, x, x, dropout=0.1)
    with pytest.raises(ValueError, match="together"):
        d2p_amd.qk_norm_rope(x, x, cos=torch.zeros(4, 8))
    m = d2p_amd.SequenceAttention(32, 4, 2, num_buckets=8, max_distance=16)
    assert m.bias.shape == (8, 4) and m.buckets.shape == (33,)
    assert m.qkv.weight.shape == (8 * 8, 32)
    with pytest.raises(ValueError, match="causal"):
        m.step(torch.randn(1, 1, 32), m.new_cache(1, 8))
    for args, match in (((32, 5), "divide"), ((32, 4, 3), "multiple"), ((32, 0), "multiple"),
                        ((48, 4), "head_dim"), ((32, 4, 2, 136), "head_dim")):
        with pytest.raises(ValueError, match=match):
            d2p_amd.SequenceAttention(*args)


def test_philox_known_answer():
    """The published first block of the generator: zero counter, zero key, 7 rounds."""
    z = np.zeros(1, dtype=np.uint64)
    assert [int(w[0]) for w in ref.philox(z, z, z, z, 0, 0)] == \
        [0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48]


def test_oracle_gradient_against_differences():
    """The 64-bit attention the kernels are checked with, against its own differences."""
    g = torch.Generator().manual_seed(1)
    q, k, v, grad = (torch.randn(1, n, 2, 8, generator=g) for n in (5, 7, 7, 5))
    bias, where = torch.randn(3, 2, generator=g), torch.tensor([0, 2, 1, 1, 0], dtype=torch.int32)
    kw = dict(causal=True, buckets=where, drop=60, seed=4)
    res, _ = ref.attention(q, k, v, grad, bias=bias, **kw)
    for n, name in enumerate(("dq", "dk", "dv", "dbias")):
        xs = [q, k, v, bias]
        d = torch.randn(xs[n].shape, generator=g).double()

        def f(h):
            ys = [x.double() for x in xs]
            ys[n] = ys[n] + h * d
            ref.U[torch.float64] = ref.TINY[torch.float64] = 0.0
            return (ref.attention(*ys[:3], bias=ys[3], **kw)[0]["out"] * grad.double()).sum()

        h = 1e-5     # h^2 f''' / 6 and 1e-16 f / h are both below 1e-9
        assert abs((f(h) - f(-h)) / (2 * h) - (res[name] * d).sum()) < 1e-8


def test_forward_mode_raises():
    """No operator has a derivative in forward mode: a tangent raises, on whichever input, and is
    never dropped (meta tensors: the operators' autograd layer without their kernels)."""
    import torch.autograd.forward_ad as fwd
    m = dict(device="meta")
    q, k = torch.empty(2, 5, 4, 16, **m), torch.empty(2, 7, 2, 16, **m)
    bias, where = torch.empty(3, 4, **m), torch.empty(5, dtype=torch.int32, **m)
    w, cos = torch.empty(16, **m), torch.empty(5, 8, **m)

    def attend(q, k, v, b):
        return d2p_amd.attention(q, k, v, bias=b, buckets=where)

    def norm(q, k, wq, wk, c, s):
        return d2p_amd.qk_norm_rope(q, k, wq, wk, c, s)

    for f, args in ((attend, (q, k, k, bias)), (norm, (q, q[:, :, :2], w, w, cos, cos))):
        f(*args)
        for n, x in enumerate(args):
            def of(y):
                return f(*args[:n], y, *args[n + 1:])
            with pytest.raises(RuntimeError, match="forward AD"):
                torch.func.jvp(of, (x,), (torch.ones_like(x),))
            for grad in (False, True):
                with fwd.dual_level(), pytest.raises(RuntimeError, match="forward AD"):
                    of(fwd.make_dual(x.detach().requires_grad_(grad), torch.ones_like(x)))
        with torch.no_grad(), fwd.dual_level(), pytest.raises(RuntimeError, match="forward AD"):
            of(fwd.make_dual(x, torch.ones_like(x)))
        # nor has the backward pass
        x = args[0].detach().requires_grad_()
        out = f(x, *args[1:])
        out = out if isinstance(out, torch.Tensor) else out[0]
        g = torch.ones_like(out)
        torch.autograd.grad(out, x, g, retain_graph=True)
        with fwd.dual_level(), pytest.raises(RuntimeError, match="forward AD"):
            torch.autograd.grad(out, x, fwd.make_dual(g, g))


def test_layer_tables_stay_in_32_bits():
    """Rotation tables are float32 whatever type the layer is moved to, and unrounded."""
    want = d2p_amd.rope_tables(50, 8, 100.0)
    for moves in ((torch.bfloat16,), (torch.float16, torch.float32), (torch.float64, torch.bfloat16)):
        m = d2p_amd.SequenceAttention(32, 4, num_buckets=8, max_length=50, rope_base=100.0)
        for to in moves:
            m = m.to(to)
        assert m.qkv.weight.dtype == m.bias.dtype == moves[-1] and m.buckets.dtype == torch.int32
        assert all(a.dtype == torch.float32 and torch.equal(a, b) for a, b in zip((m.cos, m.sin), want))
