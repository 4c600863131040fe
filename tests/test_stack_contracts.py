"""What the operators around the attention layers promise without a GPU: layouts that a compiled
program plans with, what a graph keeps, and refusals."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import d2p_amd
from test_stack_host import FAKE, HEADER, lib, residual, said  # noqa: F401


def sources(device):
    """(a source of clipping, whether its memory is dense)"""
    a = torch.ones(40, 30, device=device)
    return ((a, True), (a.t(), True), (a.view(2, 20, 30).permute(2, 0, 1), True), (a[:1], True),
            (a[:, ::2], False), (a[:, ::2].t(), False), (a[5:, 3:], False), (a[:, 1:2].t(), False),
            (a[:1].expand(9, 30), False), (a.view(2, 20, 30)[:, ::3].permute(2, 1, 0), False),
            (a[:0], True), (a[0, 0], True))


def test_fakes_of_clipped_tensors_have_the_operators_strides():
    """Sources in dense memory keep its order, others are answered with contiguous memory."""
    with FakeTensorMode():
        ts = sources("cuda")
        got, _ = d2p_amd.clip_gradients([t for t, _ in ts], 1.0)
        for r, (t, dense) in zip(got, ts):
            assert r.shape == t.shape
            assert r.stride() == (t.stride() if dense else torch.empty(t.shape).stride()), t.stride()


def kept(f):
    """The tensors that the graph of f() keeps."""
    got = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: got.append(t) or t, lambda t: t):
        out = f()
    return got, out


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.float32, torch.float16),
                                   (torch.bfloat16, torch.bfloat16)], ids=str)
def test_a_stream_without_norms_keeps_what_its_gradients_read(types):
    """(Meta tensors: the operators' autograd layer without their kernels.)"""
    x, y, gate = (torch.empty(2, 5, 16, device="meta", dtype=t, requires_grad=True)
                  for t in (types[0], types[1], types[1]))
    op = d2p_amd.residual_norm
    got, (h, _) = kept(lambda: op(x, y, norm=None, scale=0.5))
    assert not got
    dx, dy = torch.autograd.grad(h, (x, y), torch.empty_like(h))
    assert (dx.dtype, dy.dtype) == types and dx.shape == dy.shape == x.shape
    got, (h, _) = kept(lambda: op(x, y, norm=None, gate=gate))     # y and the gate
    assert len(got) == 2 and all(t.shape == x.shape and t.dtype == types[1] for t in got)
    grads = torch.autograd.grad(h, (x, y, gate), torch.empty_like(h))
    assert [g.dtype for g in grads] == [types[0], types[1], types[1]]
    got, (h, _) = kept(lambda: op(x, y, norm=None, gate=gate.detach()))
    assert len(got) == 1
    torch.autograd.grad(h, (x, y), torch.empty_like(h))
    got, (h, _) = kept(lambda: op(x, y, norm=None, post_norm="rms"))
    assert sorted(t.shape[-1] for t in got) == [4, 16]              # y and its norm's statistics
    torch.autograd.grad(h, (x, y), torch.empty_like(h))
    got, (h, n) = kept(lambda: op(x, y))
    assert sum(t.shape == x.shape for t in got) == (1 if types[0] == torch.float32 else 2)
    torch.autograd.grad((h, n), (x, y), (torch.empty_like(h), torch.empty_like(n)))


def test_statistics_are_aligned_in_both_directions(lib):  # noqa: F811
    """The forward pass writes what the backward pass reads: one rule, in the header too."""
    p = ctypes.byref(residual())
    for at in (0x1004, 0x1008):
        assert lib.d2p_residual_norm(p, FAKE, FAKE, FAKE, FAKE, ctypes.c_void_p(at), None) == 1
        assert "aligned" in said(lib)
    assert "aligned to 16 bytes" in open(HEADER).read()


def caches_that_do_not_fit(m, batch=2):
    """(tokens that come, caches, what is said)"""
    good = m.new_caches(batch, 8)
    return ((3, good[:1], "cache for each"), (3, [], "cache for each"),
            (3, good[:1] + [m.layers[1].new_cache(batch, 2)], "do not fit"),
            (3, good[:1] + [m.layers[1].new_cache(batch + 1, 8)], "sequences"),
            (9, good, "do not fit"))


def test_steps_check_every_cache_first():
    m = d2p_amd.SequenceEncoder(5, 16, 2, 2, causal=True)
    for n, caches, match in caches_that_do_not_fit(m):
        with pytest.raises(ValueError, match=match):
            m.step(torch.zeros(2, n, dtype=torch.int64), caches)
    with pytest.raises(ValueError, match="tokens must"):
        m.step(torch.zeros(2, dtype=torch.int64), m.new_caches(2, 8))
    with pytest.raises(ValueError, match="causal"):
        m = d2p_amd.SequenceEncoder(5, 16, 2, 2)
        m.step(torch.zeros(2, 1, dtype=torch.int64), m.new_caches(2, 8))


def test_the_operator_gives_no_result_that_is_not_there():
    """None in its place, with gradients as without: not a tensor of no numbers that a program could
    take a gradient of.  (Meta tensors: the operators' autograd layer without their kernels.)"""
    op = torch.ops.d2p_amd.residual_norm
    x, y = (torch.empty(2, 5, 16, device="meta", requires_grad=True) for _ in range(2))
    first = (None, None, None, None, None, None, 1, 0, 1.0, 1.0, 1e-6, torch.float32)
    plain = (None, None, None, None, None, 0, 0, 1.0, 1.0, 1e-6, torch.float32)
    for grad in (True, False):
        with torch.set_grad_enabled(grad):
            h, n = op(x, *first)
            assert h is None and n.shape == x.shape and n.requires_grad == grad
            h, n = op(x, y, *plain)
            assert n is None and h.shape == x.shape and h.requires_grad == grad
