"""GPU: the softmax of fp32 operands is as accurate as fp32 for classes far below the largest logit.  Every logit is exact here.  In units of
2^-24 of a class's share: the exponentials (of the segment's largest and of the class's logit relative to it) are off by at most 4 each and the
sum of them by 12 (an exponential, and 8 levels of additions), the quotient, the products and the terms' sum by 8: 28; and as many again for the
column's sum of 2 to 7 rows."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,classes,limit", [(128, 700, None), (1600, 700, None), (128, 700, 1)])
def test_small_shares(built, rows, classes, limit):
    import torch
    import tf_approximate_b200 as ax
    labels = torch.arange(rows, device="cuda") % 64
    x = torch.zeros(rows, 64, device="cuda")
    x[torch.arange(rows), labels] = 1.0
    w = torch.zeros(64, classes, device="cuda")
    w[:, 64:] = -torch.linspace(1.0, 70.0, classes - 64, device="cuda")
    w[:, :64] = -80.0
    w[torch.arange(64), torch.arange(64)] = 0.0
    b = torch.zeros(classes, device="cuda")
    _, _, _, db = ax.dense_cross_entropy_gradients(x, w, labels, b, reduction="sum", scratch_limit=limit)
    p = torch.softmax((x.double() @ w.double()), 1).sum(0)[64:]
    assert bool(((db[64:].double() - p).abs() <= p * 56 * 2.0 ** -24).all())
