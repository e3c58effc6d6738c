"""GPU: GELU and its slope for 16-bit results, far into the tail where the result is small.  The kernel's Phi(z) is good to 2^-17 of
itself, and z^2 / 2 in the exponent, 72 at most here, is off by a few 2^-24 of itself, which is 2^-15 of the result: 2^-13 is asked for, beside one
rounding (and half of the type's smallest step)."""
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
STEP = {"bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 2, 40, 300])
def test_gelu_keeps_its_relative_accuracy(built, rows, dtype):
    import torch
    import tf_approximate_b200 as ax
    dt = getattr(torch, dtype)
    z = torch.linspace(-12.0, 12.0, 4096, device="cuda").to(dt)
    w = torch.zeros(z.numel(), 16, device="cuda", dtype=dt)                   # units, inputs: one row of x is read with either kernel
    w[:, 0] = z
    x = torch.zeros(rows, 16, device="cuda", dtype=dt)
    x[:, 0] = 1.0
    y, kept = ax.dense_forward(x, w.t(), None, None, "gelu")
    assert torch.equal(kept, z.expand(rows, -1))
    zd = z.double()
    upper, bell = 0.5 * torch.special.erfc(-zd * 0.5 ** 0.5), torch.exp(-0.5 * zd * zd) * 0.3989422804014327
    want = zd * upper
    assert bool(((y.double() - want).abs() <= want.abs() * (UNIT[dtype] + 2.0 ** -13) + STEP[dtype]).all())
    _, _, _, dz = ax.dense_backward(torch.ones_like(y), x, w.t(), kept, "gelu", residual=y)
    slope = upper + zd * bell
    assert bool(((dz.double() - slope).abs() <= slope.abs() * UNIT[dtype] + (upper + zd.abs() * bell) * 2.0 ** -13 + STEP[dtype]).all())
