"""What test_dropout_recomputation.py checks on the CPU and test_gpu_dropout_recomputation.py on the GPU: a layer whose forward pass runs again in the
backward pass (torch.utils.checkpoint) has the same mask in both."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint


def the_gradients_mask_is_the_outputs(device, reentrant, capturable):
    import tf_approximate_b200 as ax
    layer = ax.Dropout(0.5, seed=3, capturable=capturable).to(device)
    x = torch.rand(2000, device=device).add_(0.5).requires_grad_()
    w = torch.ones(2000, device=device, requires_grad=True)
    for step in range(3):
        x.grad = w.grad = None
        y = checkpoint(lambda v: layer(v) * w, x, use_reentrant=reentrant)
        y.sum().backward()
        kept = y.detach() != 0
        assert torch.equal(x.grad != 0, kept) and torch.equal(w.grad != 0, kept)
        assert int(layer.calls) == step + 1                   # recomputation is no call of its own
        assert torch.equal(y.detach(), ax.dropout(x.detach(), 0.5, 3, step) * w.detach())


def segments_and_calls_in_any_order(device, reentrant, capturable):
    """One layer several times in a segment, two segments, two batches under way at once, random numbers drawn between."""
    import tf_approximate_b200 as ax
    layer, plain = [ax.Dropout(0.3, seed=8, capturable=capturable).to(device) for _ in range(2)]
    start = torch.rand(500, device=device).add_(0.5)
    def network(drop, x, run):
        def segment(v):
            v = drop(v) + v
            torch.rand(3)
            return drop(v * v) + drop(v)
        return run(segment, run(segment, x))
    grads = []
    for drop, run in ((layer, lambda f, v: checkpoint(f, v, use_reentrant=reentrant)), (plain, lambda f, v: f(v))):
        leaves = [start.clone().requires_grad_() for _ in range(2)]
        outs = [network(drop, v, run) for v in leaves]
        for out in outs:
            out.sum().backward()
        grads.append([v.grad for v in leaves])
        assert int(drop.calls) == 12
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def a_state_that_is_not_preserved_is_refused(device, reentrant):
    import tf_approximate_b200 as ax
    layer = ax.Dropout(0.5, seed=3).to(device)
    x = torch.rand(100, device=device, requires_grad=True)
    y = checkpoint(lambda v: layer(v) * x, x, use_reentrant=reentrant, preserve_rng_state=False)
    torch.rand(1)
    with pytest.raises(ax.InvalidArgumentError):
        y.sum().backward()
    y = layer(x)                                              # and the layer is as it was
    y.sum().backward()
    assert layer.calls == 2


def the_same_seed_of_torch_twice_makes_two_masks(device):
    import tf_approximate_b200 as ax
    layer, x, masks = ax.Dropout(0.5, seed=3), torch.ones(1000, device=device, requires_grad=True), []
    for step in range(2):
        torch.manual_seed(1)
        y = checkpoint(layer, x, use_reentrant=False)
        assert torch.equal(y.detach(), ax.dropout(x.detach(), 0.5, 3, step))
        assert torch.equal(torch.autograd.grad(y.sum(), x)[0], y.detach())
