"""What the operators around the attention layers promise: layouts, memory kept, calls that a
documented use leads to."""
import pytest
import torch

import d2p_amd
from test_stack_contracts import sources

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
