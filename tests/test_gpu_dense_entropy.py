"""GPU: the cross entropy of a dense classifier and its gradients against 64 bits, with the exponentials kept and in pieces of the
classes, rows without a label, masked classes, extreme logits, and its refusals.

Bounds.  A logit is off by sum_error(inputs) S, S = |x| |kernel| + |bias|; the largest of a row's, e, bounds the loss's error and the
relative error of the softmax (2 e) beside 2^-19 of the exponentials' own.  The gradient of a logit is rounded once to 16 bits (kept
bf16: after its exponential was rounded to fp16, 2^-12 of it or 2^-25 of the segment's largest), and the products add sum_error."""
import pytest

from test_gpu_dense import TINY, UNIT, sum_error

pytestmark = pytest.mark.gpu

SIZES = [(1, 1, 1), (1, 64, 1000), (3, 8, 10), (64, 64, 10), (130, 72, 65), (257, 136, 1000), (100, 1030, 129), (515, 64, 4099), (300, 40, 20000)]


def make(t, k, v, dtype, order, ignored=0.2, scale=1.0, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + t + k + v)
    dt = getattr(torch, dtype)
    x = (torch.randn(t, k, device="cuda", generator=g) * scale).to(dt)
    w = (torch.randn((k, v) if order == "in_out" else (v, k), device="cuda", generator=g) * k ** -0.5).to(dt)
    labels = torch.randint(v, (t,), device="cuda", generator=g)
    labels = torch.where(torch.rand(t, device="cuda", generator=g) < ignored, torch.full_like(labels, -100), labels)
    return x, w if order == "in_out" else w.t(), torch.randn(v, device="cuda", generator=g).to(dt), labels


def check_entropy(x, w, b, labels, dtype, reduction="mean", scale=1.0, limit=None):
    import torch
    import tf_approximate_b200 as ax
    u, tiny = UNIT[dtype], TINY[dtype]
    loss, dx, dw, db = ax.dense_cross_entropy_gradients(x, w, labels, b, reduction=reduction, grad_scale=scale, scratch_limit=limit, check=True)
    xd, wd = x.double(), w.double()
    logits = xd @ wd + (b.double() if b is not None else 0.0)
    valid = labels != -100
    count = max(1, int(valid.sum())) if reduction == "mean" else 1
    lse = torch.logsumexp(logits, 1)
    at = labels.clamp(min=0)
    rows = torch.where(valid, lse - logits.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    size = xd.abs() @ wd.abs() + (torch.where(torch.isfinite(b), b, torch.zeros_like(b)).double().abs() if b is not None else 0.0)
    e = size.amax(1) * sum_error(x.shape[1], dtype) + (logits.abs().nan_to_num(0.0, 0.0, 0.0).amax(1) + 1) * 2.0 ** -22     # per row
    off_row = 2 * e + 2.0 ** -19
    got_loss, got_rows = ax.dense_cross_entropy(x, w, labels, b, reduction=reduction, row_losses=True, scratch_limit=limit)
    assert torch.equal(got_loss, loss)
    assert bool(((got_rows.double() - rows).abs() <= off_row).all())
    assert abs(float(loss) - float(rows.sum()) / count) <= float((off_row * valid).sum()) / count + 2.0 ** -20 * float(rows.sum()) / count + 1e-30
    p = torch.exp(logits - lse[:, None])
    d = p.clone()
    d[torch.arange(len(labels), device="cuda"), at] -= 1.0
    d *= (valid.double() / count * scale)[:, None]
    share = (valid.double() / count * scale)[:, None]
    off = p * share * (2 * e[:, None] + 2.0 ** -18)
    if dtype != "float32":
        off += u * d.abs() * (1 + 2.0 ** -4) + tiny * share / 16384.0 * (dtype == "float16")
        off += p * share * 2.0 ** -11 + share * 2.0 ** -24        # the kept exponential's rounding
    else:
        off += 2.0 ** -22 * d.abs()
    off += 1e-40                                                  # the smallest value of bf16, which a stored gradient is made of
    for got, want, s, o, depth in ((dx, d @ wd.t(), d.abs() @ wd.t().abs(), off @ wd.t().abs(), w.shape[1]),
                                   (dw, xd.t() @ d, xd.t().abs() @ d.abs(), xd.t().abs() @ off, x.shape[0])):
        assert got.shape == want.shape and got.dtype == x.dtype
        assert bool(((got.double() - want).abs() <= o + s * sum_error(depth, dtype) * 1.01 + want.abs() * u + tiny).all())
    if b is not None:
        bt = str(b.dtype)[6:]
        assert bool(((db.double() - d.sum(0)).abs() <= off.sum(0) + len(labels) * 2.0 ** -23 * d.abs().sum(0) + UNIT[bt] * d.sum(0).abs() + TINY[bt]).all())
    else:
        assert db is None


@pytest.mark.parametrize("limit", [None, 1])
@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("t,k,v", SIZES)
def test_sizes(built, t, k, v, dtype, order, limit):
    """limit 1: pieces of 256 classes, the most of them."""
    x, w, b, labels = make(t, k, v, dtype, order)
    check_entropy(x, w, b if (t + v) % 2 else None, labels, dtype, ("mean", "sum")[t % 2], 256.0 if dtype == "float16" else 1.0, limit)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_few_pieces(built, dtype):
    """Pieces that neither the classes nor the tiles divide evenly."""
    x, w, b, labels = make(200, 64, 5000, dtype, "in_out")
    for classes in (1024, 3000):
        check_entropy(x, w, b, labels, dtype, limit=200 * classes * (6 if dtype == "float32" else 2))


@pytest.mark.parametrize("rows,limit", [(140, None), (140, 1), (1600, None)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_extreme_logits_and_masked_classes(built, dtype, rows, limit):
    """Few logits, pieces of the classes, kept exponentials."""
    import torch
    import tf_approximate_b200 as ax
    x, w, b, labels = make(rows, 64, 700, dtype, "in_out", scale=100.0)      # logits of some hundreds
    check_entropy(x, w, b, labels, dtype, limit=limit)
    low = float(torch.finfo(b.dtype).min)
    for masked in (float("-inf"), low):
        b2 = b.clone()
        b2[64:200] = masked                                                 # whole segments of 64 classes and parts of some
        b2[699] = masked
        lab = torch.where((labels >= 64) & (labels < 200) | (labels == 699), torch.zeros_like(labels), labels)
        check_entropy(x, w, b2, lab, dtype, limit=limit)
        loss, dx, dw, db = ax.dense_cross_entropy_gradients(x, w, lab, b2, scratch_limit=limit)
        assert bool((dw[:, 64:200] == 0).all()) and bool((db[64:200] == 0).all()) and bool(torch.isfinite(dx).all())


@pytest.mark.parametrize("rows,limit", [(77, None), (77, 1), (4000, None)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_rows_without_label(built, dtype, rows, limit):
    import torch
    import tf_approximate_b200 as ax
    x, w, b, labels = make(rows, 40, 300, dtype, "out_in")
    for reduction in ("mean", "sum"):
        loss, dx, dw, db = ax.dense_cross_entropy_gradients(x, w, torch.full_like(labels, -100), b, reduction=reduction, scratch_limit=limit)
        assert float(loss) == 0.0 and not bool(dx.any()) and not bool(dw.any()) and not bool(db.any())
        loss, dx, dw, db = ax.dense_cross_entropy_gradients(x[:0], w, labels[:0], b, reduction=reduction, scratch_limit=limit)
        assert float(loss) == 0.0 and dx.shape == (0, 40) and not bool(dw.any()) and not bool(db.any())
    _, dx, _, _ = ax.dense_cross_entropy_gradients(x, w, labels, b, scratch_limit=limit)
    assert bool((dx[labels == -100] == 0).all()) and bool((dx[labels != -100] != 0).any(1).all())
    other = torch.where(labels == -100, torch.full_like(labels, 299), labels)
    check = ax.dense_cross_entropy_gradients(x, w, other, b, ignore_index=299, scratch_limit=limit)[0]
    assert bool(torch.isfinite(check))


@pytest.mark.parametrize("rows,limit", [(77, None), (77, 1), (4000, None)])
def test_labels_that_are_no_class(built, rows, limit):
    import torch
    import tf_approximate_b200 as ax
    for wrong in (-1, 300, 1 << 40, -(1 << 40)):
        x, w, b, labels = make(rows, 40, 300, "bfloat16", "in_out", ignored=0.0)
        labels[5] = wrong
        loss, dx, dw, db = ax.dense_cross_entropy_gradients(x, w, labels, b, scratch_limit=limit)
        _, losses = ax.dense_cross_entropy(x, w, labels, b, row_losses=True)
        assert bool(torch.isnan(loss)) and torch.isnan(losses).nonzero()[:, 0].tolist() == [5]
        assert torch.isnan(dx).any(1).nonzero()[:, 0].tolist() == [5] and bool(torch.isnan(dw).any())


def test_logits_that_are_not_finite(built):
    import torch
    import tf_approximate_b200 as ax
    for value, count in ((float("nan"), 150), (float("inf"), 150), (float("nan"), 4000), (float("inf"), 4000)):
        x, w, b, labels = make(count, 64, 300, "bfloat16", "in_out", ignored=0.0)
        b[100] = value
        loss, rows = ax.dense_cross_entropy(x, w, labels, b, row_losses=True)
        assert not bool(torch.isfinite(loss)) and not bool(torch.isfinite(rows[labels != 100]).any())
        for limit in (None, 1):
            assert bool(torch.isnan(ax.dense_cross_entropy_gradients(x, w, labels, b, scratch_limit=limit)[1]).any())


def test_autograd_strides_and_differences(built):
    import torch
    import tf_approximate_b200 as ax
    x, w, b, labels = make(60, 48, 500, "float32", "in_out")
    explicit = ax.dense_cross_entropy_gradients(x, w, labels, b)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    loss = ax.dense_cross_entropy(leaves[0].view(5, 12, 48), leaves[1], labels.view(5, 12), leaves[2])
    (3.0 * loss).backward()
    for v, e in zip(leaves, explicit[1:]):
        assert torch.allclose(v.grad, 3.0 * e, rtol=1e-6, atol=0)
    check_entropy(x.t().contiguous().t(), w[:, 1:], b[1:], labels.clamp(max=498), "float32")
    layer = ax.Dense(48, 500).cuda()
    with torch.no_grad():
        layer.kernel.copy_(w)
        layer.bias.copy_(b)
        assert torch.equal(layer.cross_entropy(x, labels), loss.detach())
        # along the gradient: (f(p + h d) - f(p - h d)) / 2h; the loss is near 7 and off by 2^-20 of it at most
        for p, e in zip((x, w, b), explicit[1:]):
            norm = float(e.norm())
            h, d, f = 2.0 ** -5, e / e.norm(), []
            for sign in (1, -1):
                p += sign * h * d
                f.append(float(ax.dense_cross_entropy(x, w, labels, b)))
                p -= sign * h * d
            assert abs((f[0] - f[1]) / (2 * h) - norm) < 0.02 * norm + 2 * 7 * 2.0 ** -20 / (2 * h)


def test_refusals(built):
    import torch
    import tf_approximate_b200 as ax
    x, w, b, labels = make(4, 8, 16, "float32", "in_out")
    for args in ((x, w, labels.int()), (x, w, labels[:3]), (x, w, labels.cpu()), (x, w.half(), labels), (x, w[:7], labels), (x, w, labels, b[:3]),
                 (x.double(), w.double(), labels), (x, w[:, :0], labels), (x[:, :0], w[:0], labels)):
        with pytest.raises(ax.InvalidArgumentError):
            ax.dense_cross_entropy_gradients(*args)
    with pytest.raises(ax.InvalidArgumentError):
        ax.dense_cross_entropy(x, w, labels, reduction="none")
    with pytest.raises(ax.InvalidArgumentError):
        ax.Dense(4, 4, activation="relu").cuda().cross_entropy(x[:, :4], labels)
