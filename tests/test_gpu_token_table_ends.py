"""Both ways of the token table's gradient, sums in LDS and the sort, at the ends of their ranges.
Each case states the way it goes, by the workspace that the library asks for."""
import ctypes

import pytest
import torch

import d2p_amd
from test_stack_host import Embedding, Strides, lib  # noqa: F401

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
E = 2.0 ** -24


@pytest.fixture
def clean(cuda):
    torch.cuda.empty_cache()
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def sorts(lib, N, V, D):  # noqa: F811
    """Whether the library asks for keys and positions of all N tokens, twice."""
    p = Embedding(0, 2, 1, N, V, D, ctypes.c_void_p(0x1000), 4, None, -1, 1.0, Strides(N * D, D))
    need = lib.d2p_token_embedding_backward_workspace_bytes(ctypes.byref(p))
    assert need >= 16 * N or need <= 64 << 20
    return need >= 16 * N


# V: the last in LDS, the first in one pass of the sort, one of two passes, one of three
@pytest.mark.parametrize("V,way", [(64, False), (65, True), (1030, True), ((1 << 20) + 5, True)])
def test_as_many_tokens_as_there_may_be(cuda, clean, lib, V, way):  # noqa: F811
    N, D = 2 ** 31 - 1, 8
    assert sorts(lib, N, V, D) == way
    tokens = torch.empty(1, N, dtype=torch.int32, device=cuda)
    want = torch.zeros(V, dtype=torch.float64)
    for part in tokens[0].split(1 << 28):
        torch.arange(part.numel(), out=part)
        part.remainder_(V - 1)
        n = part.numel()
        want[:V - 1] += n // (V - 1) + (torch.arange(V - 1) < n % (V - 1)).double()
    for n in (5, N // 2, *range(N - 7, N)):     # the last token: at both ends, and in between
        want[int(tokens[0, n])] -= 1
        want[V - 1] += 1
        tokens[0, n] = V - 1
    assert float(want.sum()) == N and want[V - 1] == 9
    grad = torch.ones(1, 1, D, dtype=BF16, device=cuda).expand(1, N, D)
    dw = torch.ops.d2p_amd.token_embedding_backward(grad, tokens, None, 1.0, -1, V, F32).cpu().double()
    assert torch.equal(dw[V - 1], torch.full((D,), 9.0, dtype=torch.float64))
    # Sums of up to 2^24 ones are exact; others are joined from parts.  By the sort: chunks of 128
    # positions or more, taken in turn by the 256 teams that 8 features leave, then those 256 sums.
    # In LDS: at most 1024 parts and their 256 teams.  Each addition is off by E of what there is.
    joins = want / 128 / 256 + 2 + 256 if way else torch.full((V,), 1024.0 + 256)
    joins = torch.where(want <= 2 ** 24, 0.0, joins)
    assert ((dw - want[:, None]).abs() <= (want * E * joins)[:, None]).all()


def test_gradients_past_2_to_31_numbers_in_lds(cuda, clean, lib):  # noqa: F811
    V, D = 2, 6144
    L = 2 ** 31 // D + 77
    assert not sorts(lib, L, V, D) and sorts(lib, L, V, D + 8)
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, V, (1, L), generator=g).to(cuda)
    rows = torch.tensor([0, 1, L // 2, L - 90, L - 2, L - 1], device=cuda)
    grad = torch.zeros(1, L, D, dtype=BF16, device=cuda)
    grad[0, rows] = torch.randint(-9, 10, (6, D), generator=g).to(BF16).to(cuda)
    want = torch.zeros(V, D, device=cuda).index_add_(0, tokens[0, rows], grad[0, rows].float())
    for kind in (torch.int64, torch.int32):
        dw = torch.ops.d2p_amd.token_embedding_backward(grad, tokens.to(kind), None, 1.0, -1, V, F32)
        assert torch.equal(dw, want)        # sums of whole numbers
    weight = torch.randn(V, D, generator=g).to(BF16).to(cuda)
    del grad
    out = d2p_amd.token_embedding(tokens, weight)
    assert torch.equal(out[0, rows], weight[tokens[0, rows]])
