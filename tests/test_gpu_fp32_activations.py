"""GPU: activations and slopes of fp32 results are as accurate as fp32, far into the tails.  In units of 2^-24 of the result: expf, erfcf and
the division are off by at most 8 together, the operations around them by 6, and the argument's rounding (z / sqrt 2, twice in the
exponent) by 2 z^2 for GELU.  Of a slope's two parts each is that good; 1 - sigmoid is off by 2^-24 of 1."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("rows", [1, 8, 40])
@pytest.mark.parametrize("activation", ["gelu", "silu"])
def test_relative_accuracy(built, activation, rows, order):
    import torch
    import tf_approximate_b200 as ax
    z = torch.linspace(-12.0, 12.0, 4096, device="cuda")
    w = torch.zeros((16, 4096) if order == "in_out" else (4096, 16), device="cuda")
    w = w if order == "in_out" else w.t()
    w[0] = z
    x = torch.zeros(rows, 16, device="cuda")
    x[:, 0] = 1.0
    y, kept = ax.dense_forward(x, w, None, None, activation)
    k = kept.double()
    if activation == "gelu":
        below, bell = 0.5 * torch.special.erfc(-k * 0.5 ** 0.5), torch.exp(-0.5 * k * k) * 0.3989422804014327
        want, slope, parts, units = k * below, below + k * bell, below + k.abs() * bell, 14 + 2 * k * k
    else:
        s = torch.sigmoid(k)
        want, slope, parts, units = k * s, s * (1 + k * (1 - s)), s * (1 + k.abs() * (1 - s)), 14 + 0 * k
        parts = parts + s * k.abs() / units                            # 2^-24 of 1 in 1 - s
    assert bool(((y.double() - want).abs() <= want.abs() * units * 2.0 ** -24).all())
    _, _, _, dz = ax.dense_backward(torch.ones_like(y), x, w, kept, activation, residual=y)
    assert bool(((dz.double() - slope).abs() <= parts * units * 2.0 ** -24).all())
