"""GPU: gradients whose squares leave fp32's range.  Beyond it the second moment is infinite, the step m / inf = 0, and decay alone is left,
as the formula has it; below the normal numbers the root is still that of what is there."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_squares_beyond_fp32(built, dtype, bits):
    import torch
    import tf_approximate_b200 as ax
    dt = getattr(torch, dtype)
    p = torch.full((1000,), 2.0, device="cuda", dtype=dt)
    g = torch.ones(1000, device="cuda", dtype=dt)
    g[::3] = 2.0 ** 80
    g[1::6] = -2.0 ** 100
    opt = ax.AdamW([p], lr=0.25, weight_decay=0.5, state_bits=bits)
    opt.step([g])
    large = g.abs() > 2
    assert torch.equal(p[large], torch.full_like(p[large], 1.75))
    # beside them: a step of lr against the gradient's sign
    assert torch.allclose(p[~large].float(), torch.full_like(p[~large], 1.5).float(), rtol=2.0 ** -20)
    if bits == 32:
        opt.step([g])
        assert torch.equal(p[large].float(), torch.full_like(p[large], 1.75 * 0.875).float())
        assert bool(torch.isinf(opt.exp_avg_sq[:1000][large]).all()) and bool(torch.isfinite(p).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_squares_below_the_normal_numbers(built, bits):
    """(1 - beta2) g^2 = 0.001 2^-120 has 19 bits left: its root is good to 2^-20, and the first step is the learning rate."""
    import torch
    import tf_approximate_b200 as ax
    p = torch.ones(1000, device="cuda")
    g = torch.full((1000,), 2.0 ** -60, device="cuda")
    g[::2] = -g[::2]
    ax.AdamW([p], lr=0.25, eps=0.0, weight_decay=0.0, state_bits=bits).step([g])
    assert torch.allclose(p, 1.0 - 0.25 * torch.sign(g), rtol=2.0 ** -18)
