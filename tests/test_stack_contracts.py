"""What the operators around the attention layers promise without a GPU: layouts that a compiled
program plans with, what a graph keeps, and refusals."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import d2p_amd


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
