"""CPU: the dropout layer refuses in evaluation what it refuses in training."""
import pytest


def test_residuals_of_another_kind(built):
    import torch
    import tf_approximate_b200 as ax
    layer, x = ax.Dropout(0.5, seed=1).eval(), torch.randn(3, 8)
    for bad in (torch.zeros(3, 8).half(), torch.zeros(3, 8).double(), torch.zeros(8), torch.zeros(1, 8), torch.zeros(3, 8, device="meta"), 1.0):
        with pytest.raises(ax.InvalidArgumentError):
            layer(x, residual=bad)
    r = torch.randn(3, 8, requires_grad=True)
    assert layer(x) is x and torch.equal(layer(x, residual=r), x + r) and layer(x, r).requires_grad
    assert torch.equal(layer(x.t(), residual=r.t()), (x + r).t())
