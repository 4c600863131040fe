"""What the operators around the attention layers promise: layouts, memory kept, calls that a
documented use leads to."""
import ctypes

import pytest
import torch

import d2p_amd
from test_stack_contracts import caches_that_do_not_fit, sources
from test_stack_host import Residual, Strides, Vector, lib  # noqa: F401

pytestmark = pytest.mark.gpu


def test_compiled_clipping_of_any_layout(cuda):
    """A program traced with the operator's fake runs on what the operator gives."""
    for t, dense in sources(cuda):
        torch._dynamo.reset()       # (each layout a program of its own)
        eager = d2p_amd.clip_gradients([t], 2.0)[0][0]
        assert eager.stride() == (t.stride() if dense else torch.empty(t.shape).stride())
        f = torch.compile(lambda t: d2p_amd.clip_gradients([t], 2.0)[0][0].mul(2.0),
                          backend="aot_eager", fullgraph=True)
        got = f(t)
        assert got.stride() == eager.mul(2.0).stride() and torch.equal(got, 2.0 * eager)
        if not dense:       # whose numbers lie in order
            f = torch.compile(lambda t: d2p_amd.clip_gradients([t], 2.0)[0][0].view(-1),
                              backend="aot_eager", fullgraph=True)
            assert torch.equal(f(t), eager.reshape(-1))


@pytest.mark.parametrize("D", [513, 1024, 2048])
def test_a_backward_pass_fills_the_card_whatever_gradients_are_wanted(cuda, lib, D):  # noqa: F811
    """Rows of several waves: the kernel has four waves a SIMD with and without sums for the biases,
    so as many workgroups leave parts of the vectors' gradients in the workspace."""
    B, L = 2, 4096 + 7
    x, y, dh, dn = (torch.randn(B, L, D, device=cuda).bfloat16() for _ in range(4))
    w, b = torch.ones(D, device=cuda), torch.zeros(D, device=cuda)
    stats = torch.ones(B, L, 4, device=cuda)
    dx, dy = torch.empty_like(x), torch.empty_like(x)
    dw, db = torch.empty_like(w), torch.empty_like(b)
    rows = Strides(L * D, D)

    def ptr(t):
        return None if t is None else ctypes.c_void_p(t.data_ptr())

    def parts(db):
        p = Residual(2, 2, B, L, D, 1, rows, rows, rows, rows, 2, 0, Vector(ptr(w), 0), Vector(ptr(b), 0),
                     Vector(None, 0), Vector(None, 0), 0, None, 0, Strides(0, 0), 0.5, 1.0, 1e-5)
        need = lib.d2p_residual_norm_backward_workspace_bytes(ctypes.byref(p))
        ws = torch.full((need // 4,), float("nan"), device=cuda)
        assert lib.d2p_residual_norm_backward(
            ctypes.byref(p), ptr(dh), ptr(dn), ptr(x), ptr(y), ptr(stats), ptr(dx), ptr(dy), None,
            ptr(dw), ptr(db), None, None, ptr(ws), need,
            ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        torch.cuda.synchronize()
        written = int((~ws.isnan()).sum())
        assert written % D == 0
        return written // D

    assert parts(db) == 2 * parts(None)


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.float32, torch.float16),
                                   (torch.bfloat16, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("D", [8, 9, 96, 520])
def test_a_stream_without_norms_needs_no_stream_in_its_backward_pass(cuda, types, D):
    """Gradients from results' gradients alone, at any alignment; x is not kept for them."""
    g = torch.Generator().manual_seed(D)

    def whole(*shape, dtype):       # numbers whose products and sums here are exact
        return torch.randint(-4, 5, shape, generator=g).to(dtype).to(cuda)

    y = whole(2, 5, D, dtype=types[1]).requires_grad_()
    gate = whole(D, dtype=torch.float32).requires_grad_()
    for shift in (0, 1, 3):
        dh = whole(2 * 5 * D + shift, dtype=types[0])[shift:].view(2, 5, D)
        for m in (None, gate):
            x = whole(2, 5, D, dtype=types[0]).requires_grad_()
            h, n = d2p_amd.residual_norm(x, y, norm=None, gate=m, scale=0.5, residual_scale=2.0)
            assert n is None and torch.equal(h, (2 * x.float() + 0.5 * (1 if m is None else m) * y.float())
                                             .to(types[0]))
            got = torch.autograd.grad(h, [x, y] + [m] * (m is not None), dh)
            assert torch.equal(got[0], 2 * dh)
            assert torch.equal(got[1], (0.5 * (1 if m is None else m.detach()) * dh.float()).to(types[1]))
            if m is not None:
                assert torch.equal(got[2], (0.5 * dh.float() * y.detach().float()).sum((0, 1)))


def test_a_refused_step_leaves_the_caches(cuda):
    m = d2p_amd.SequenceEncoder(5, 16, 2, 2, causal=True).to(cuda)
    for n, caches, match in caches_that_do_not_fit(m):
        with pytest.raises(ValueError, match=match):
            m.step(torch.zeros(2, n, dtype=torch.int64, device=cuda), caches)
        assert not any(t.any() for c in caches for t in c)
    caches = m.new_caches(2, 8) + m.new_caches(2, 8)        # more than there are layers
    m.step(torch.zeros(2, 1, dtype=torch.int64, device=cuda), caches)
    assert [int(c.lengths[0]) for c in caches] == [1, 1, 0, 0]


@pytest.mark.parametrize("dtype,other", [(torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16)])
def test_a_16_bit_encoder_under_autocast_to_the_other_16_bits(cuda, dtype, other):
    """The stream keeps its type, the blocks run in autocast's: within 30 roundings of bfloat16, the
    coarser of the two, of the encoder in 32 bits."""
    torch.manual_seed(0)
    m = d2p_amd.SequenceEncoder(23, 64, 4, 3, 2, causal=True, post_norm="rms", gated=0.3).to(cuda).eval()
    tokens = torch.randint(0, 23, (3, 40), device=cuda)
    want = m(tokens)
    m = m.to(dtype)
    with torch.autocast("cuda", dtype=other):
        got = m(tokens)
        got.float().square().sum().backward()
        caches = m.new_caches(3, 40)
        steps = torch.cat([m.step(tokens[:, a:b], caches) for a, b in ((0, 9), (9, 10), (10, 40))], 1)
    assert got.dtype == steps.dtype == dtype
    assert all(p.grad.dtype == dtype and p.grad.isfinite().all() for p in m.parameters())
    for out in (got, steps):
        assert (out - want).abs().max() <= 30 * 2.0 ** -8 * want.abs().max()


def test_lengths_that_pass_32_bits_are_wrong_ones(cuda):
    """They come back NaN as other lengths out of range do, in the layer and in the encoder."""
    m = d2p_amd.SequenceEncoder(23, 64, 4, 2).to(cuda)
    tokens = torch.randint(0, 23, (4, 12), device=cuda)
    lengths = torch.tensor([12, 2 ** 32 + 12, -2 ** 32 + 5, 7], device=cuda)
    for out in (m(tokens, lengths), m.layers[0](torch.randn(4, 12, 64, device=cuda), lengths)):
        assert out[1:3].isnan().all() and out[::3].isfinite().all()
    assert torch.equal(m(tokens, lengths)[::3], m(tokens, lengths.clamp(0, 12).int())[::3])


def test_results_in_another_order_share_no_memory_either(cuda):
    """Refused before anything is written, as results in their source's order are."""
    op = d2p_amd.clip_gradients
    base = torch.zeros(64, device=cuda)
    x, y = torch.ones(6, 5, device=cuda), torch.ones(10, device=cuda)
    turned = base[:30].view(5, 6).t()
    for out in ([turned, base[29:39]], [turned, base[:10]], [turned, y[:1].expand(10)]):
        with pytest.raises(RuntimeError, match="share|single memory"):
            op([x, y], 1.0, out=out)
        with pytest.raises(RuntimeError, match="share|single memory"):
            op([y, x], 1.0, out=out[::-1])
    with pytest.raises(RuntimeError, match="share"):
        op([x, x.clone()], 1.0, out=[turned, base[:30].view(5, 6).t()])
    # a gradient that is broadcast: the others are not clipped when it is refused
    p, q = (torch.nn.Parameter(torch.zeros(4, 4, device=cuda)) for _ in range(2))
    p.grad, q.grad = torch.ones(4, 4, device=cuda), torch.ones(1, 1, device=cuda).expand(4, 4)
    with pytest.raises(RuntimeError, match="single memory"):
        d2p_amd.clip_grad_norm_([p, q], 1.0)
    assert not base.any() and (p.grad == 1).all() and (x == 1).all() and (y == 1).all()
    # what stays apart is written: neighbours, columns of one buffer, a source's own memory turned
    want, _ = op([x, y], 1.0)
    op([x, y], 1.0, out=[turned, base[30:40]])
    assert torch.equal(turned, want[0]) and torch.equal(base[30:40], want[1]) and not base[40:].any()
    columns = torch.zeros(10, 2, device=cuda)
    got, _ = op([y, 2 * y], 1.0, out=[columns[:, 0], columns[:, 1]])
    assert torch.equal(columns[:, 1], 2 * columns[:, 0]) and columns.all()
    empty = torch.ones(1, 1, device=cuda).expand(4, 4)[:0]      # of no numbers: nothing is written
    op([empty, y], 1.0, out=[empty, base[30:40]])
    a = torch.arange(16.0, device=cuda).view(4, 4)
    want, _ = op([a.t()], 1.0)
    op([a.t()], 1.0, out=[a])
    assert torch.equal(a, want[0])


def test_operators_registrations_agree(cuda):
    """Schemas, fakes, autograd and compiled programs, as torch's own check has it.  (Clipped results
    share one buffer, which that check does not allow.)"""
    o = torch.ops.d2p_amd
    t = torch.randint(0, 9, (3, 7), device=cuda)
    w = torch.randn(9, 16, device=cuda, requires_grad=True)
    lengths = torch.tensor([7, 2, 0], dtype=torch.int32, device=cuda)
    x, y = (torch.randn(3, 7, 16, device=cuda, requires_grad=True) for _ in range(2))
    v = torch.randn(16, device=cuda, requires_grad=True)
    ts = [torch.randn(5, device=cuda), torch.randn(4, 6, device=cuda).t(),
          torch.randn(4, 6, device=cuda)[:, ::2]]
    into = [torch.empty(a.shape, device=cuda) for a in ts]
    for op, args in ((o.token_embedding, (t, w, lengths, 2.0, 3, torch.float16)),
                     (o.residual_norm, (x, y, v, v, v, v, v, 2, 2, 0.5, 1.0, 1e-6, torch.float32)),
                     (o.residual_norm, (x, y, *[None] * 5, 0, 0, 0.5, 1.0, 1e-6, torch.float32)),
                     (o.residual_norm, (x, None, v, *[None] * 4, 1, 0, 1.0, 1.0, 1e-6, torch.bfloat16)),
                     (o.global_norm, (ts,)), (o.clip_gradients_into, (ts, 1.0, into))):
        torch.library.opcheck(op.default, args)


def test_second_derivative_without_norms_raises(cuda):
    x, y = (torch.randn(2, 5, 32, device=cuda, requires_grad=True) for _ in range(2))
    g = torch.randn(2, 5, 32, device=cuda, requires_grad=True)
    h, _ = d2p_amd.residual_norm(x, y, norm=None, scale=0.5)
    d = torch.autograd.grad(h, (x, y), g, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        d[1].sum().backward()
