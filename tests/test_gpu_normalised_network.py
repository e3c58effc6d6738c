"""GPU: table convolutions, group norm with activation and shortcut, dropout, the dense head and its cross entropy in one training step against 64 bits,
and the same network answering in 8 bits (with examples/retrain_classifier.py)."""
import importlib.util
import os

import pytest

import philox

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load_example():
    spec = importlib.util.spec_from_file_location("retrain_classifier", os.path.join(ROOT, "examples", "retrain_classifier.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    return example


def test_a_training_step_against_64_bits(built):
    """From the convolution's output on every operator is exact, so that the step has a reference; the convolution itself has its own tests, and
    its kernel's gradient here is the exact convolution's of the gradient that reaches it."""
    import torch
    import tf_approximate_b200 as ax
    torch.manual_seed(3)
    conv = ax.FakeApproxConv2D(8, 24, 3, padding="same", mul_map_file=ax.Table(array=ax.noisy_table(3001))).cuda()
    norm, again = ax.GroupNorm(24, 6, activation="silu").cuda(), ax.GroupNorm(24, 4, activation="gelu").cuda()
    drop, head = ax.Dropout(0.3, seed=77), ax.Dense(24, 10).cuda()
    x, labels = torch.randn(16, 9, 11, 8, device="cuda"), torch.randint(10, (16,), device="cuda")
    features = conv(x)
    features.retain_grad()
    hidden = norm(features)
    mixed = again(drop(hidden), residual=features)
    loss = head.cross_entropy(mixed.mean((1, 2)), labels)
    loss.backward()
    f, ns, no, gs, go, hk, hb = [t.detach().double().requires_grad_() for t in (features, norm.scale, norm.offset, again.scale, again.offset, head.kernel, head.bias)]
    F = torch.nn.functional
    def group_norm(v, groups, s, o):
        return F.group_norm(v.permute(0, 3, 1, 2), groups, s, o, 1e-3).permute(0, 2, 3, 1)
    h = F.silu(group_norm(f, 6, ns, no))
    keep = torch.from_numpy(philox.keep(0, h.numel(), 0.3, 77, 0)).cuda().view(h.shape)
    h = torch.where(keep, h * (65536 / (65536 - philox.share(0.3))), torch.zeros_like(h))
    want = F.cross_entropy(F.gelu(group_norm(h, 4, gs, go) + f).mean((1, 2)) @ hk + hb, labels)
    want.backward()
    # fp32 throughout: sums of some 10^4 values whose terms are off by a few 2^-24
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5
    for got, ref in ((features.grad, f.grad), (norm.scale.grad, ns.grad), (norm.offset.grad, no.grad), (again.scale.grad, gs.grad), (again.offset.grad, go.grad),
                     (head.kernel.grad, hk.grad), (head.bias.grad, hb.grad)):
        assert float((got.double() - ref).norm() / ref.norm()) < 2e-5
    assert conv.kernel.grad is not None and bool(conv.kernel.grad.isfinite().all()) and float(conv.kernel.grad.abs().max()) > 0
    # the step that follows takes another mask
    assert drop.calls == 1 and not torch.equal(drop(hidden.detach()) == 0, ~keep)


def test_the_example_with_all_of_them(built):
    import torch
    example = load_example()
    losses, right = example.train(steps=3, batch=64, groups=8, dropout=0.1, answer_8bit=True)
    assert len(losses) == 3 and all(v == v and 0 < v < 100 for v in losses) and 0.0 <= right <= 1.0
    import tf_approximate_b200 as ax
    torch.manual_seed(0)
    net = example.Classifier(ax.Table(array=ax.noisy_table(3001)), groups=8, dropout=0.1).cuda().eval()
    images = torch.randn(40, 16, 16, 3, device="cuda")
    with torch.no_grad():
        exact = net(images)
    answer = net.in_8bit()(images)
    # codes have three bits behind the leading one: operands are off by 2^-4 of themselves at most, their products' sums by less than a tenth in all
    assert float((answer - exact).norm() / exact.norm()) < 0.1
