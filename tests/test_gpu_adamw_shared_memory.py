"""GPU: parameters that share memory are refused, neighbours in one buffer are not."""
import pytest

pytestmark = pytest.mark.gpu


def test_parameters_that_share_memory(built):
    import torch
    import tf_approximate_b200 as ax
    flat = torch.zeros(1000, device="cuda")
    for params in ([flat, flat.detach()], [flat[:500], flat[499:]], [flat[10:20], flat], [flat.view(10, 100), flat[3:4]]):
        with pytest.raises(ax.InvalidArgumentError):
            ax.AdamW(params)
    parts = [flat[500:], flat[:0], flat[:300], flat[300:500], flat[300:300]]
    ax.AdamW(parts, lr=0.5, weight_decay=0.0).step([torch.ones_like(p) for p in parts])
    assert torch.allclose(flat, torch.full_like(flat, -0.5))
