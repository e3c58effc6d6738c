"""GPU: tensors whose memory holds the other sign (the imaginary part of a conjugate) are read as the values that they stand for, and refused as
parameters."""
import pytest

pytestmark = pytest.mark.gpu


def test_negative_views(built):
    import torch
    import tf_approximate_b200 as ax
    g = torch.Generator(device="cuda").manual_seed(0)
    view = lambda *s: torch.randn(*s, device="cuda", dtype=torch.complex64, generator=g).conj().imag  # noqa: E731
    x, w, b, r, dy = view(20, 16), view(16, 12), view(12), view(20, 12), view(20, 12)
    assert x.is_neg()
    plain = [t.resolve_neg().clone() for t in (x, w, b, r, dy)]
    y, kept = ax.dense_forward(x, w, b, r, "silu")
    want, want_kept = ax.dense_forward(*plain[:4], "silu")
    assert torch.equal(y, want)
    for a, e in zip(ax.dense_backward(dy, x, w, kept, "silu", bias=b, residual=r), ax.dense_backward(plain[4], *plain[:2], want_kept, "silu", bias=plain[2], residual=plain[3])):
        assert torch.equal(a, e)
    labels = torch.randint(12, (20,), device="cuda", generator=g)
    for a, e in zip(ax.dense_cross_entropy_gradients(x, w, labels, b), ax.dense_cross_entropy_gradients(*plain[:2], labels, plain[2])):
        assert torch.equal(a, e)
    p, q = torch.zeros(20, 16, device="cuda"), torch.zeros(20, 16, device="cuda")
    ax.AdamW([p]).step([x])
    ax.AdamW([q]).step([plain[0]])
    assert torch.equal(p, q)
    opt = ax.AdamW([p])
    opt.params[0] = torch.zeros(20, 16, device="cuda")._neg_view()
    with pytest.raises(ax.InvalidArgumentError):
        opt.step([plain[0]])
