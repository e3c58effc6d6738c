"""GPU: dropout against its definition: the mask to the bit, kept values within one rounding of fp32 and one of the type."""
import pytest

import philox

pytestmark = pytest.mark.gpu

UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def check_dropout(x, rate, seed, offset, residual=None, where=None):
    import torch
    import tf_approximate_b200 as ax
    y = ax.dropout(x, rate, seed, offset, residual) if where is None else ax.dropout(x, rate, seed, where, residual)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    keep = torch.from_numpy(philox.keep(0, x.numel(), rate, seed, offset)).cuda().view(x.shape)
    share = philox.share(rate)
    part = x.double() * (65536 / (65536 - share) if share < 65536 else 0.0)
    want = torch.where(keep, part, torch.zeros_like(part))
    r = torch.zeros_like(want) if residual is None else residual.double()
    u = UNIT[str(x.dtype)[6:]]
    # the factor and the product are rounded to fp32, and the sum with the residual
    assert bool(((y.double() - (want + r)).abs() <= 3 * 2.0 ** -24 * (want.abs() + r.abs()) + u * (want + r).abs() + 2.0 ** -25).all())
    if residual is None:
        assert bool((y[~keep] == 0).all()) and bool((y[keep & (x != 0)] != 0).all())
    return y


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (256, 2048), (1001, 777), (4096,), (4097,), (2, 3, 5, 17)])
def test_sizes(built, shape, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(len(shape))
    x, r = [torch.randn(shape, device="cuda", generator=g).to(getattr(torch, dtype)) for _ in range(2)]
    for rate, seed, offset in ((0.5, 1, 0), (0.1, 0xffffffffffffffff, 0xfedcba9876543210), (0.9, 1 << 32, 1 << 32)):
        check_dropout(x, rate, seed, offset)
        check_dropout(x, rate, seed, offset, r)


def test_rates_at_the_ends(built):
    import torch
    import tf_approximate_b200 as ax
    x = torch.randn(5000, device="cuda")
    assert torch.equal(ax.dropout(x, 0.0, 3), x) and torch.equal(ax.dropout(x, 2.0 ** -18, 3), x)
    for rate in (1.0, 1 - 2.0 ** -18):
        y = ax.dropout(x, rate, 3)
        assert bool((y == 0).all())
        assert torch.equal(ax.dropout(x, rate, 3, residual=x), x)
    check_dropout(x, 2.0 ** -16, 3, 0)
    check_dropout(x, 1 - 2.0 ** -16, 3, 0)
    # what is dropped is 0 whatever it was
    bad = torch.full((4096,), float("nan"), device="cuda")
    keep = torch.from_numpy(philox.keep(0, 4096, 0.3, 9)).cuda()
    y = ax.dropout(bad, 0.3, 9)
    assert bool(y[keep].isnan().all()) and bool((y[~keep] == 0).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides_and_alignment(built, dtype):
    import torch
    dt = getattr(torch, dtype)
    def rand(*s):
        return torch.randn(*s, device="cuda").to(dt)
    views = [rand(40, 30).t(), rand(30, 80)[:, ::2], rand(1201)[1:].view(30, 40), rand(1204)[4:].view(30, 40), rand(1, 40).expand(30, 40), rand(30, 47)[:, 3:43]]
    for i, x in enumerate(views):
        check_dropout(x, 0.4, 11, 5)
        check_dropout(x, 0.4, 11, 5, views[i - 1])


def test_the_mask_depends_on_place_seed_and_offset_alone(built):
    import torch
    import tf_approximate_b200 as ax
    one = torch.ones(3000, device="cuda")
    a = ax.dropout(one, 0.5, 7, 3)
    assert torch.equal(a, ax.dropout(one.bfloat16(), 0.5, 7, 3).float()) and torch.equal(a[:1001], ax.dropout(one[:1001], 0.5, 7, 3))
    for seed, offset in ((8, 3), (7, 4), (7 + (1 << 32), 3), (7, 3 + (1 << 32))):
        b = ax.dropout(one, 0.5, seed, offset)
        agree = float((a == b).float().mean())
        assert abs(agree - 0.5) < 5 * 0.5 / 3000 ** 0.5          # five deviations of 3000 fair coins


def test_more_values_than_31_bits_count(built):
    import numpy as np
    import torch
    import tf_approximate_b200 as ax
    n = (1 << 31) + 1003
    x = torch.ones(n, dtype=torch.float16, device="cuda")
    y = ax.dropout(x, 0.25, 5, 6)
    first = (1 << 31) - 4000
    keep = philox.keep(first, n - first, 0.25, 5, 6)
    assert np.array_equal(y[first:].cpu().numpy() != 0, keep)
    assert abs(float((y == 0).sum(dtype=torch.int64)) / n - 0.25) < 5 * (0.25 * 0.75 / n) ** 0.5


def test_gradients(built):
    import torch
    import tf_approximate_b200 as ax
    x, r = [torch.randn(37, 50, device="cuda", requires_grad=True) for _ in range(2)]
    g = torch.randn(37, 50, device="cuda", requires_grad=True)
    y = ax.dropout(x, 0.3, 21, 4, residual=r)
    dx, dr = torch.autograd.grad(y, (x, r), g, create_graph=True)
    assert torch.equal(dx, ax.dropout(g, 0.3, 21, 4)) and torch.equal(dr, g)
    # linear: the gradient's gradient is the same mask once more
    h = torch.randn_like(g)
    assert torch.equal(torch.autograd.grad(dx, g, h)[0], ax.dropout(h, 0.3, 21, 4))
    d = torch.randn_like(x)
    with torch.no_grad():
        slope = (ax.dropout(x + d, 0.3, 21, 4).double() - ax.dropout(x, 0.3, 21, 4).double())
    assert float((slope - ax.dropout(d, 0.3, 21, 4).double()).abs().max()) < 1e-5
    y = ax.dropout(x, 0.3, 21, 4)
    assert torch.equal(torch.autograd.grad(y, x, g.detach())[0], ax.dropout(g.detach(), 0.3, 21, 4))


def test_offsets_on_the_device(built):
    import torch
    import tf_approximate_b200 as ax
    x = torch.randn(1000, device="cuda", requires_grad=True)
    where = torch.tensor((5 << 32) + 7, device="cuda")
    y = check_dropout(x.detach(), 0.5, 3, (5 << 32) + 7, where=where)
    assert torch.equal(y, ax.dropout(x.detach(), 0.5, 3, (5 << 32) + 7))
    z = ax.dropout(x, 0.5, 3, where)
    where.add_(1)
    with pytest.raises(RuntimeError):            # the counter moved on: the mask of the forward pass is gone
        z.sum().backward()


def test_captured_steps(built):
    """The layer: another mask at every replay, the same one in both passes of a replay.  (x is this graph's own leaf: no eager graph of it lives.)"""
    import torch
    import tf_approximate_b200 as ax
    x = torch.randn(1000, device="cuda", requires_grad=True)
    layer = ax.Dropout(0.5, seed=17, capturable=True).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(layer(x).sum(), x)
        layer.calls.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = layer(x)
            dx, = torch.autograd.grad(out.sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    for call in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert int(layer.calls) == call + 1
        assert torch.equal(out.detach(), ax.dropout(x.detach(), 0.5, 17, call)) and torch.equal(dx, ax.dropout(torch.ones_like(x), 0.5, 17, call))


def test_layer(built):
    import torch
    import tf_approximate_b200 as ax
    x, r = torch.randn(64, 32, device="cuda"), torch.randn(64, 32, device="cuda")
    layer = ax.Dropout(0.25, seed=5)
    assert torch.equal(layer(x), ax.dropout(x, 0.25, 5, 0)) and torch.equal(layer(x, residual=r), ax.dropout(x, 0.25, 5, 1, r))
    layer.eval()
    assert layer(x) is x and torch.equal(layer(x, residual=r), x + r) and layer.calls == 2
    assert ax.Dropout(0.25).seed != ax.Dropout(0.25).seed
    assert ax.dropout(torch.zeros(0, 5, device="cuda"), 0.5, 1).shape == (0, 5)


def test_refusals(built):
    import torch
    import tf_approximate_b200 as ax
    x = torch.randn(8, device="cuda")
    for call in (lambda: ax.dropout(x, 1.01, 1), lambda: ax.dropout(x, -0.01, 1), lambda: ax.dropout(x, float("nan"), 1), lambda: ax.dropout(x, 0.5, -1), lambda: ax.dropout(x, 0.5, 1 << 64),
                 lambda: ax.dropout(x, 0.5, 1.0), lambda: ax.dropout(x, 0.5, 1, -1), lambda: ax.dropout(x, 0.5, 1, torch.zeros(2, dtype=torch.int64, device="cuda")),
                 lambda: ax.dropout(x, 0.5, 1, torch.zeros((), dtype=torch.int32, device="cuda")), lambda: ax.dropout(x, 0.5, 1, torch.zeros((), dtype=torch.int64)),
                 lambda: ax.dropout(x.double(), 0.5, 1), lambda: ax.dropout(x, 0.5, 1, residual=x[:4]), lambda: ax.dropout(x, 0.5, 1, residual=x.half())):
        with pytest.raises(ax.InvalidArgumentError):
            call()
