"""GPU: fp32 products with infinities: inf times a finite value is an infinity of their signs' product, inf times zero and sums of both
infinities are NaN, and nothing else changes, in the forward product and in both gradients."""
import pytest

pytestmark = pytest.mark.gpu


def product(a, b):
    """sum over k of a[m, k] b[k, n], product by product in 64 bits"""
    return (a.double()[:, :, None] * b.double()[None]).sum(1)


def same(got, want):
    import torch
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf] > 0, want[inf] > 0)
    fine = torch.isfinite(want)
    # values near 1, sums of at most 300 products of them: the sums are off by less than 2^-16 of 300
    assert bool(((got[fine].double() - want[fine]).abs() < 300 * 2.0 ** -16).all())


@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("t,k,n", [(40, 64, 24), (33, 300, 136), (260, 20, 20), (12, 130, 257)])
def test_infinities_in_either_operand(built, t, k, n, order):
    import torch
    import tf_approximate_b200 as ax
    inf = float("inf")
    g = torch.Generator(device="cuda").manual_seed(t + k + n)
    x = torch.randn(t, k, device="cuda", generator=g)
    w = torch.randn((k, n) if order == "in_out" else (n, k), device="cuda", generator=g)
    w = w if order == "in_out" else w.t()
    w[:, 1] = 1.0                                          # whole in one bf16 term
    w[3, 5:8] = torch.tensor([0.0, -0.0, 1e-30], device="cuda")
    dy = torch.randn(t, n, device="cuda", generator=g)
    for place in ("x", "kernel", "both", "opposite", "gradient"):
        x2, w2, dy2 = x.clone(), w.clone(), dy.clone()
        if place in ("x", "both", "opposite"):
            x2[4, 3], x2[7, 9] = inf, -inf
        if place in ("kernel", "both"):
            w2[3, 11], w2[10, 2] = inf, -inf
        if place == "opposite":
            x2[4, 11] = -inf
        if place == "gradient":
            dy2[2, 3], dy2[9, 1] = -inf, inf
            x2[2, 6] = 0.0
        same(ax.dense(x2, w2), product(x2, w2))
        dx, dw, db, _ = ax.dense_backward(dy2, x2, w2, bias=w2[0].clone())
        same(dx, product(dy2, w2.t()))
        same(dw, product(x2.t(), dy2))
        assert torch.equal(torch.isinf(db), torch.isinf(dy2).any(0))


def test_infinite_gradient_through_an_activation(built):
    """The output's gradient is split after the activation's slope."""
    import torch
    import tf_approximate_b200 as ax
    g = torch.Generator(device="cuda").manual_seed(0)
    x, w, dy = (torch.randn(*s, device="cuda", generator=g) for s in ((50, 16), (16, 36), (50, 36)))
    y, kept = ax.dense_forward(x, w, None, None, "relu")
    row, column = (y > 0).nonzero()[5].tolist()
    dy[row, column] = float("inf")
    dx, dw, _, _ = ax.dense_backward(dy, x, w, kept, "relu")
    dz = torch.where(y > 0, dy, torch.zeros_like(dy))
    same(dx, product(dz, w.t()))
    same(dw, product(x.t(), dz))
