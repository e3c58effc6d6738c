"""GPU: the layer's masks when a forward pass is run again in the backward pass."""
import pytest

import dropout_recomputed as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("capturable", [False, True])
def test_recomputation(built, reentrant, capturable):
    R.the_gradients_mask_is_the_outputs("cuda", reentrant, capturable)
    R.segments_and_calls_in_any_order("cuda", reentrant, capturable)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_state_that_is_not_preserved(built, reentrant):
    R.a_state_that_is_not_preserved_is_refused("cuda", reentrant)


def test_the_same_seed_of_torch_twice(built):
    R.the_same_seed_of_torch_twice_makes_two_masks("cuda")


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputation_in_a_captured_step(built, reentrant):
    """Another mask at every replay, the same one in both passes.  (x is this graph's own leaf: no eager graph of it lives.)"""
    import torch
    from torch.utils.checkpoint import checkpoint
    import tf_approximate_b200 as ax
    layer = ax.Dropout(0.5, seed=17, capturable=True).cuda()
    x, got = torch.rand(1000, device="cuda").add_(0.5).requires_grad_(), torch.zeros(1000, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = checkpoint(layer, x, use_reentrant=reentrant)
            y.sum().backward()
            got.copy_(x.grad)
            x.grad = None
    torch.cuda.current_stream().wait_stream(side)
    for call in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert int(layer.calls) == call + 1
        assert torch.equal(y.detach(), ax.dropout(x.detach(), 0.5, 17, call)) and torch.equal(got, ax.dropout(torch.ones(1000, device="cuda"), 0.5, 17, call))
