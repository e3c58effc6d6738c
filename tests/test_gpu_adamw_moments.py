"""GPU: moments that are not the tensors that the optimizer made are refused before anything is launched."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_replaced_moments_are_refused(built, bits):
    import torch
    import tf_approximate_b200 as ax
    p = torch.ones(600, device="cuda")
    opt = ax.AdamW([p], state_bits=bits)
    names = ("exp_avg", "exp_avg_sq") if bits == 32 else ("exp_avg", "exp_avg_sq_root", "exp_avg_scale", "exp_avg_sq_root_scale")
    for name in names:
        kept = getattr(opt, name)
        for other in (kept.cpu(), kept[:1], kept.view(torch.uint8), torch.zeros(2 * kept.numel(), device="cuda").to(kept.dtype)[::2], None):
            setattr(opt, name, other)
            with pytest.raises(ax.InvalidArgumentError):
                opt.step([torch.ones_like(p)])
        setattr(opt, name, kept.clone())           # another tensor of the same kind is fine
    assert opt.step_count == 0 and bool((p == 1).all())
    opt.step([torch.ones_like(p)])
    assert opt.step_count == 1 and bool((p < 1).all())
