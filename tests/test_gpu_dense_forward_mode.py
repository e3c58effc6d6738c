"""GPU: forward-mode differentiation is refused, as it is where a gradient is asked for; it is not dropped."""
import pytest

from test_gpu_dense_entropy import make

pytestmark = pytest.mark.gpu


def test_dual_numbers_are_refused(built):
    import torch
    import torch.autograd.forward_ad as forward_ad
    import tf_approximate_b200 as ax
    x, w, b, labels = make(30, 16, 20, "float32", "in_out")
    plain, loss = ax.dense(x, w, b), ax.dense_cross_entropy(x, w, labels, b)
    for grad in (False, True):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            for at in range(3):
                operands = [forward_ad.make_dual(v, torch.ones_like(v)) if i == at else v for i, v in enumerate((x, w, b))]
                with pytest.raises(RuntimeError):
                    ax.dense(*operands)
                with pytest.raises(RuntimeError):
                    ax.dense_cross_entropy(operands[0], operands[1], labels, operands[2])
            # tensors without a tangent are served as ever
            assert torch.equal(ax.dense(x, w, b), plain) and torch.equal(ax.dense_cross_entropy(x, w, labels, b), loss)
