"""CPU: what is no tensor is refused with the package's own error, whether or not a gradient may be asked for."""
import numpy as np
import pytest


@pytest.mark.parametrize("grad", [False, True])
def test_operands_that_are_no_tensors(built, grad):
    import torch
    import tf_approximate_b200 as ax
    w, labels = torch.zeros(3, 4, requires_grad=grad), torch.zeros(2, dtype=torch.int64)
    for x in (None, 1.0, [[0.0] * 3] * 2, np.zeros((2, 3), np.float32)):
        for call in (lambda: ax.dense(x, w), lambda: ax.dense(w, x), lambda: ax.dense(w, w, x if x is not None else 1), lambda: ax.dense_cross_entropy(x, w, labels),
                     lambda: ax.dense_cross_entropy(w, x, labels), lambda: ax.dense_cross_entropy(w, w, x), lambda: ax.dense_forward(x, w), lambda: ax.dense_backward(x, w, w)):
            with pytest.raises(ax.InvalidArgumentError):
                call()
