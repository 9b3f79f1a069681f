"""The direct route of the rotary embedding: which captured backward passes it refuses, and what it takes as sections."""

import contextlib
import gc

import pytest
import torch

from tests.test_gpu_rotary import _check, _freqs, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("direct", [True, False])
def test_a_leaf_that_is_not_reached_may_be_held(direct):
    """An eager graph from the default stream holds the query; the captured pass computes the keys' gradient alone."""
    import torch_neuronx_b200 as T
    from torch_neuronx_b200 import _lib

    if _lib.native is None:
        pytest.skip("the check is part of the direct entry points")
    g = torch.Generator().manual_seed(8)
    q, k = (torch.randn(2, 5, h, 64, generator=g).transpose(1, 2) for h in (4, 2))
    gk = torch.randn(2, 2, 5, 64, generator=g)
    pos, freq = torch.randint(0, 300, (2, 5), generator=g), _freqs(64)
    lq, lk = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    dk, dp, df = gk.cuda(), pos.cuda(), freq.cuda()

    def step():
        with contextlib.nullcontext() if direct else torch.device("cuda"):
            yq, yk = T.rotary_embedding(lq, lk, dp, df)
            return torch.autograd.grad((yq, yk), (lk,), (yq.detach(), dk))[0]

    alive = T.rotary_embedding(lq, None, dp, df)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    side.synchronize()
    dk.neg_()
    graph.replay()
    torch.cuda.synchronize()
    _check(got.detach().cpu(), _want(-gk, pos.expand(1, 2, 5), freq, (32,), False, -1.0))
    assert alive[0].grad_fn is not None
    del alive
    gc.collect()


def test_sections_of_a_list_take_the_direct_route():
    """A model's configuration holds a list."""
    from torch_neuronx_b200 import _lib

    if _lib.native is None:
        pytest.skip("there is no direct route")
    q, pos, freq = torch.randn(1, 2, 5, 64, device="cuda"), torch.arange(15, device="cuda").view(3, 1, 5), _freqs(64).cuda()
    with torch._C.DisableTorchFunction():
        got = [_lib.native.rotary(q, None, pos, freq, s, False) for s in ((8, 12, 12), [8, 12, 12])]
        assert got[1] is not None and torch.equal(got[0][0], got[1][0])
        assert _lib.native.rotary(q, None, pos, freq, [8, 12, "12"], False) is None and _lib.native.rotary(q, None, pos, freq, [8, 24], False) is None
