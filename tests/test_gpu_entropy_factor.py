"""GPU: the factor that comes from above in the backward pass of the cross entropy is fp32, whatever the operands' type."""
import pytest

from test_gpu_dense_entropy import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,factor", [("bfloat16", 1.0 / 3.0), ("bfloat16", 0.1), ("float16", 65536.0), ("float16", 1.0 / 3.0), ("float32", 1.0 / 3.0)])
@pytest.mark.parametrize("order", ["in_out", "out_in"])
def test_gradients_are_rounded_once(built, dtype, factor, order):
    import torch
    import tf_approximate_b200 as ax
    x, w, b, labels = make(70, 48, 90, dtype, order, ignored=0.3)
    explicit = ax.dense_cross_entropy_gradients(x, w, labels, b)[1:]
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    (ax.dense_cross_entropy(leaves[0], leaves[1], labels, leaves[2]) * factor).backward()
    scale = torch.tensor(factor, dtype=torch.float32, device="cuda")
    for leaf, e in zip(leaves, explicit):
        want = (e.float() * scale).to(e.dtype)
        assert torch.isfinite(want).all() and torch.equal(leaf.grad, want) and leaf.grad.dtype == e.dtype
    assert not bool(leaves[0].grad[labels == -100].any())
