"""GPU: a gradient has its parameter's shape."""
import pytest

pytestmark = pytest.mark.gpu


def test_gradients_of_another_shape_are_refused(built):
    import torch
    import tf_approximate_b200 as ax
    p = torch.zeros(4, 6, device="cuda")
    opt = ax.AdamW([p])
    for shape in ((6, 4), (24,), (4, 6, 1), (2, 12)):
        with pytest.raises(ax.InvalidArgumentError):
            opt.step([torch.ones(*shape, device="cuda")])
    assert opt.step_count == 0 and not bool(p.any())
    opt.step([torch.ones(6, 4, device="cuda").t()])
    assert bool((p < 0).all())
