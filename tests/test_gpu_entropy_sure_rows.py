"""GPU: rows that are classified all but surely.  The label's logit is 1024 and the others are 1008, so that with s = (classes - 1) exp(-16)
the loss is log(1 + s) and the gradient of the label's logit -s / (1 + s).  Every logit is exact; the sum 1 + s is off by one rounding of 2^-24
for each of at most 40 additions and by the exponentials' own 2^-18 of s; the loss and the gradient must not be off by more, however large the logits are."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,classes,limit", [(40, 50, None), (40, 700, None), (1600, 700, None), (140, 700, 1), (1600, 1500, 1)])
def test_small_losses(built, rows, classes, limit, dtype):
    import torch
    import tf_approximate_b200 as ax
    dt = getattr(torch, dtype)
    labels = (torch.arange(rows, device="cuda") * 7) % min(classes, 64)
    x = torch.zeros(rows, 64, device="cuda", dtype=dt)
    x[torch.arange(rows), labels] = 32.0
    w = torch.full((64, classes), 31.5, device="cuda", dtype=dt)              # 32 * 31.5 = 1008
    at = torch.arange(min(classes, 64), device="cuda")
    w[at, at] = 32.0                                                          # 1024
    b = torch.zeros(classes, device="cuda")
    s = (classes - 1) * math.exp(-16.0)
    want, off = math.log1p(s), 40 * 2.0 ** -24 + 2.0 ** -18 * s
    loss, losses = ax.dense_cross_entropy(x, w, labels, b, row_losses=True, scratch_limit=limit)
    assert float((losses.double() - want).abs().max()) <= off
    assert abs(float(loss) - want) <= off + 2.0 ** -22 * want
    total, _, _, db = ax.dense_cross_entropy_gradients(x, w, labels, b, reduction="sum", scratch_limit=limit)
    # a class that rows have as their label: each of them gives -s / (1 + s), every other row exp(-16) / (1 + s)
    n = torch.bincount(labels, minlength=classes)
    want_db = (-n * s + (rows - n) * math.exp(-16.0)).double() / (1 + s)
    unit = {"float32": 2.0 ** -22, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -10}[dtype]           # the stored gradient, and the kept exponential
    off_db = n * off + (n * s + (rows - n) * math.exp(-16.0)) * (unit + 2.0 ** -18) + rows * 2.0 ** -24 * math.exp(-16.0)
    assert bool(((db.double() - want_db).abs() <= off_db).all())
