"""GPU: group norm and its gradients against 64 bits: sizes with every kind of plan, types, activations, layouts, edges.

Bounds.  D = 2^-24.  A group's mean is off by at most K D of its largest value, its variance (a sum of squares less the mean) and r by K D of
themselves; K counts the additions that a value goes through: 4 of a chunk, one for each of a thread's chunks, one for each entry that a
lane joins, 5 of the lanes, 8 of the cluster (64 holds for the sizes here but the largest, which say theirs).  z = (x - mean) r scale + offset +
residual has five roundings on top.  The activations' slopes are below 1.13, their second derivatives below 0.8, their own errors below
2^-20 of their argument (2^-17 for 16-bit results).  dx of 16-bit types is made of dz as it is rounded to them: half a step of dz more.  Sums of dz are off by K D of the sum of magnitudes and by what dz is off."""
import pytest

pytestmark = pytest.mark.gpu

D = 2.0 ** -24
UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-44, "bfloat16": 1e-40, "float16": 2.0 ** -25}
# (samples, places..., channels), groups
SHAPES = [((1, 1, 8), 1), ((2, 3), 3), ((2, 3), 1), ((1, 8, 8, 64), 8), ((3, 5, 7, 20), 4), ((2, 9, 120), 24), ((4, 33, 165), 33), ((2, 31, 31, 36), 1), ((5, 4, 4, 2048), 32),
          ((2, 700, 48), 48), ((2, 27, 45, 120), 24), ((1, 56, 56, 256), 32), ((3, 50, 1001), 7), ((2, 41, 4100), 1), ((1, 12, 5003), 1), ((300, 1, 64), 4), ((1, 1, 1, 1), 1)]
LARGE = [((2, 160, 160, 128), 32), ((1, 300, 301, 33), 3), ((1, 20000, 520), 2), ((2, 500, 2500), 1), ((1, 70000, 7), 7)]


def exact_activation(z, name):
    import torch
    F = torch.nn.functional
    return {None: lambda v: v * 1.0, "relu": torch.relu, "gelu": F.gelu, "silu": F.silu}[name](z)


def make(shape, dtype, params=None, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    dt, c = getattr(torch, dtype), shape[-1]
    def rand(*s):
        return torch.randn(*s, device="cuda", generator=g)
    x = (rand(*shape) * torch.exp(0.5 * rand(c)) + rand(c)).to(dt)
    p = getattr(torch, params or dtype)
    return x, (1 + 0.3 * rand(c)).to(p), (0.3 * rand(c)).to(p), rand(*shape).to(dt), rand(*shape).to(dt)


def check_norm(x, groups, scale, offset, residual, act, grad, epsilon=1e-3, k=64):
    import torch
    import tf_approximate_b200 as ax
    dtype = str(x.dtype)[6:]
    u, tiny, own = UNIT[dtype], TINY[dtype], (2.0 ** -20 if dtype == "float32" else 2.0 ** -17) if act else 0.0
    y, statistics = ax.group_norm_forward(x, groups, scale, offset, residual, act, epsilon)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous() and statistics.shape == (x.shape[0], groups, 2)
    n, c = x.shape[0], x.shape[-1]
    each, e = c // groups, k * D
    def parts(t):
        return t.double().reshape(n, -1, groups, each)
    xd = parts(x)
    one, zero = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    s, o = [t.double().view(1, 1, groups, each) for t in (one if scale is None else scale, zero if offset is None else offset)]
    r_ = parts(residual) if residual is not None else torch.zeros_like(xd)
    var, mean = torch.var_mean(xd, (1, 3), correction=0, keepdim=True)
    r = 1 / torch.sqrt(var + epsilon)
    off_mean = e * xd.abs().amax((1, 3), keepdim=True)
    xhat = (xd - mean) * r
    off_xhat = r * off_mean + (e + 4 * D) * xhat.abs()
    assert bool(((statistics[..., 0].double() - mean[:, 0, :, 0]).abs() <= off_mean[:, 0, :, 0] + 1e-44).all())
    assert bool(((statistics[..., 1].double() / r[:, 0, :, 0] - 1).abs() <= e + r[:, 0, :, 0] ** 2 * off_mean[:, 0, :, 0] ** 2).all())
    z = xhat * s + o + r_
    off_z = off_xhat * s.abs() + 4 * D * (z.abs() + o.abs() + r_.abs())
    want = exact_activation(z, act)
    assert bool(((parts(y) - want).abs() <= 1.13 * off_z + own * z.abs() + u * want.abs() + tiny).all())
    if grad is None:
        return
    dx, ds, do, dr = ax.group_norm_backward(grad, x, statistics, groups, scale, offset, residual, act)
    gd = parts(grad)
    zz = z.detach().requires_grad_()
    slope = (z > 0).double() if act == "relu" else torch.autograd.grad(exact_activation(zz, act).sum(), zz)[0] if act else torch.ones_like(z)
    off_slope = 0.8 * off_z + own * (1 + z.abs()) if act else torch.zeros_like(z)
    if act == "relu":                    # where z is within its error of zero either slope is one
        off_slope = (z.abs() <= off_z).double()
    dz = gd * slope
    off_dz = gd.abs() * off_slope + 2 * D * dz.abs()
    m = xd.shape[1] * each
    m1, m2 = (dz * s).sum((1, 3), keepdim=True) / m, (dz * s * xhat).sum((1, 3), keepdim=True) / m
    off1 = ((off_dz + e * dz.abs()) * s.abs()).sum((1, 3), keepdim=True) / m
    off2 = ((off_dz * xhat.abs() + dz.abs() * (off_xhat + e * xhat.abs())) * s.abs()).sum((1, 3), keepdim=True) / m
    want = r * (dz * s - m1 - xhat * m2)
    off = r * (off_dz * s.abs() + off1 + xhat.abs() * off2 + off_xhat * m2.abs() + (e + 6 * D) * (dz.abs() * s.abs() + m1.abs() + xhat.abs() * m2.abs()))
    off = off + r * s.abs() * (u * dz.abs() + tiny)          # dz, rounded to the tensors' type on its way
    assert bool(((parts(dx) - want).abs() <= off + u * want.abs() + tiny).all())
    if scale is not None:
        us = UNIT[str(scale.dtype)[6:]]
        want = (dz * xhat).sum((0, 1)).flatten()
        off = (off_dz * xhat.abs() + dz.abs() * off_xhat + (2 * e + n * D) * (dz * xhat).abs()).sum((0, 1)).flatten()
        assert ds.dtype == scale.dtype and bool(((ds.double() - want).abs() <= off + us * want.abs() + TINY[str(scale.dtype)[6:]]).all())
    if offset is not None:
        uo = UNIT[str(offset.dtype)[6:]]
        want, off = dz.sum((0, 1)).flatten(), (off_dz + (2 * e + n * D) * dz.abs()).sum((0, 1)).flatten()
        assert do.dtype == offset.dtype and bool(((do.double() - want).abs() <= off + uo * want.abs() + TINY[str(offset.dtype)[6:]]).all())
    assert (ds is None) == (scale is None) and (do is None) == (offset is None) and (dr is None) == (residual is None)
    if residual is not None:
        assert dr.shape == x.shape and bool(((parts(dr) - dz).abs() <= off_dz + u * dz.abs() + tiny).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_sizes(built, shape, groups, dtype):
    which = sum(shape) + groups
    x, scale, offset, residual, grad = make(shape, dtype, "float32" if which % 2 else dtype)
    check_norm(x, groups, scale, offset, residual if which % 3 else None, (None, "silu", "gelu", "relu")[which % 4], grad)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape,groups", LARGE)
def test_spans_that_no_cluster_holds(built, shape, groups, dtype):
    x, scale, offset, residual, grad = make(shape, dtype)
    check_norm(x, groups, scale, offset, residual if shape[0] == 2 else None, "silu", grad, k=1024)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
def test_activations_with_every_addition(built, act, dtype):
    for shape in ((3, 6, 10, 48), (2, 17, 21)):
        x, scale, offset, residual, grad = make(shape, dtype)
        for s in (scale, None):
            for o in (offset, None):
                for r in (residual, None):
                    check_norm(x, 3, s, o, r, act, grad)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides_and_alignment(built, dtype):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    def rand(*s):
        return torch.randn(*s, device="cuda", generator=g).to(dt)
    n, h, w, c = 3, 5, 9, 40
    count = n * h * w * c
    grad = rand(n, h, w, c)
    views = [rand(n, c, h, w).permute(0, 2, 3, 1), rand(n, h, w, 2 * c)[..., ::2], rand(count + 1)[1:].view(n, h, w, c), rand(count + 4)[4:].view(n, h, w, c),
             rand(n, h, w + 3, c)[:, :, 1:w + 1], rand(1, h, w, c).expand(n, h, w, c)]
    for i, x in enumerate(views):
        for r in (None, views[i - 1]):
            check_norm(x, 8, rand(2 * c)[::2], rand(c + 1)[1:], r, "silu", grad if i % 2 else views[i - 2])


def test_values_far_from_zero(built):
    """A mean that is 4096 times the spread: squares less the square of the mean would have lost the variance."""
    import torch
    for shape, groups in (((2, 30, 30, 64), 8), ((2, 160, 160, 128), 32), ((2, 77, 45), 9)):
        x, scale, offset, residual, grad = make(shape, "float32")
        check_norm(x + 4096.0, groups, scale, offset, None, "silu", grad, k=64 if shape[1] < 100 else 256)


def test_one_outlier_does_not_hide_the_others(built):
    import torch
    import tf_approximate_b200 as ax
    x = torch.randn(2, 64, 64, 32, device="cuda") * 1e-3
    x[0, 0, 0, 0] = x[1, 63, 63, 31] = 1e3
    check_norm(x, 4, None, None, None, None, torch.randn_like(x))


def test_groups_without_spread_and_values_that_are_none(built):
    import torch
    import tf_approximate_b200 as ax
    x = torch.full((2, 6, 6, 16), 3.25, device="cuda")
    y, statistics = ax.group_norm_forward(x, 4, epsilon=1e-3)
    assert bool((y == 0).all()) and bool((statistics[..., 0] == 3.25).all())
    x = torch.randn(3, 6, 6, 16, device="cuda")
    clean = ax.group_norm(x, 4)
    for bad in (float("inf"), float("nan"), -float("inf")):
        z = x.clone()
        z[1, 2, 3, 5] = bad                      # sample 1, group 1
        y = ax.group_norm(z, 4)
        mask = torch.zeros(3, 6, 6, 16, dtype=torch.bool, device="cuda")
        mask[1, :, :, 4:8] = True
        assert bool(y[mask].isnan().all()) and torch.equal(y[~mask], clean[~mask])


def test_empty(built):
    import torch
    import tf_approximate_b200 as ax
    for shape in ((0, 4, 4, 8), (3, 0, 8)):
        x = torch.zeros(shape, device="cuda")
        y, statistics = ax.group_norm_forward(x, 2, torch.ones(8, device="cuda"), torch.zeros(8, device="cuda"))
        assert y.shape == x.shape
        dx, ds, do, _ = ax.group_norm_backward(x, x, statistics, 2, torch.ones(8, device="cuda"), torch.zeros(8, device="cuda"))
        assert dx.shape == x.shape and bool((ds == 0).all()) and bool((do == 0).all())


def test_autograd_and_the_layer(built):
    import torch
    import tf_approximate_b200 as ax
    torch.manual_seed(0)
    layer = ax.GroupNorm(24, 6, activation="gelu").cuda()
    with torch.no_grad():
        layer.scale.normal_()
        layer.offset.normal_()
    x, r = torch.randn(2, 5, 6, 24, device="cuda", requires_grad=True), torch.randn(2, 5, 6, 24, device="cuda", requires_grad=True)
    g = torch.randn(2, 5, 6, 24, device="cuda")
    y = layer(x, residual=r)
    y.backward(g)
    xd, rd, sd, od = [t.detach().double().requires_grad_() for t in (x, r, layer.scale, layer.offset)]
    z = torch.nn.functional.group_norm(xd.permute(0, 3, 1, 2), 6, sd, od, 1e-3).permute(0, 2, 3, 1) + rd
    torch.nn.functional.gelu(z).backward(g.double())
    for a, b in ((x, xd), (r, rd), (layer.scale, sd), (layer.offset, od)):
        assert float((a.grad.double() - b.grad).abs().max()) < 1e-5 * (1 + float(b.grad.abs().max()))
    # against differences: a step along each gradient's direction
    step = 1e-2
    with torch.no_grad():
        for t in (x, r, layer.scale, layer.offset):
            d = t.grad / t.grad.norm()
            keep = t.detach().clone()
            t.copy_(keep + step * d)
            up = (layer(x, residual=r).double() * g).sum()
            t.copy_(keep - step * d)
            down = (layer(x, residual=r).double() * g).sum()
            t.copy_(keep)
            slope = float(up - down) / (2 * step)
            # third derivatives along a unit direction times step^2, and the fp32 rounding of 1440 values over 2 step
            assert abs(slope - float(t.grad.norm())) < 1e-2 * (1 + float(t.grad.norm()))
    x2 = torch.randn(1, 24, device="cuda")
    assert ax.GroupNorm(24, 6, use_scale=False, use_offset=False)(x2).shape == x2.shape
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(layer(x).sum(), x, create_graph=True)[0].sum(), x)


def test_the_same_every_time_and_in_a_graph(built):
    import torch
    import tf_approximate_b200 as ax
    for shape, groups in (((4, 28, 28, 64), 16), ((2, 160, 160, 128), 32)):
        x, scale, offset, residual, grad = make(shape, "bfloat16", "float32")
        def step():
            y, statistics = ax.group_norm_forward(x, groups, scale, offset, residual, "silu")
            return (y, *ax.group_norm_backward(grad, x, statistics, groups, scale, offset, residual, "silu"))
        first = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                held = step()
        torch.cuda.current_stream().wait_stream(side)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            for a, b, c in zip(first, held, step()):
                assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("shape,groups", [((2, 1100000, 1024), 2), ((70001, 8, 8, 512), 16)])
def test_more_values_than_31_bits_count(built, shape, groups):
    """Both forms beyond 2^31 values: the last sample against 64 bits (its last places, where it has many), and the statistics of all."""
    import torch
    import tf_approximate_b200 as ax
    c = shape[-1]
    x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_()
    scale, offset = torch.rand(c, device="cuda") + 0.5, torch.randn(c, device="cuda")
    y, statistics = ax.group_norm_forward(x, groups, scale, offset, None, "relu")
    last = x[-1].view(-1, groups, c // groups)
    mean = torch.stack([part.double().sum((0, 2)) for part in last.split(1 << 18)]).sum(0) / (last.shape[0] * last.shape[2])
    var = torch.stack([(part.double() - mean[:, None]).square().sum((0, 2)) for part in last.split(1 << 18)]).sum(0) / (last.shape[0] * last.shape[2])
    r = 1 / torch.sqrt(var + 1e-3)
    # means of normal values: K D times the largest, below 6, as for the other sizes
    assert float((statistics[-1, :, 0].double() - mean).abs().max()) < 1024 * D * 6 and float((statistics[-1, :, 1].double() / r - 1).abs().max()) < 1024 * D
    tail = last[-2000:].double()
    want = torch.relu(((tail - mean[:, None]) * r[:, None]).reshape(-1, c) * scale.double() + offset.double())
    got = y[-1].reshape(-1, c)[-2000:].double()
    assert bool(((got - want).abs() <= 1024 * D * 8 + UNIT["float16"] * want.abs() + TINY["float16"]).all())
    dx = ax.group_norm_backward(x, x, statistics, groups, scale, offset, None, "relu")[0]
    # the group's gradient has no part along its mean: S1 takes it out
    sums = torch.stack([part.double().sum((0, 2)) for part in dx[-1].view(-1, groups, c // groups).split(1 << 18)]).sum(0)
    assert float(sums.abs().max()) / (last.shape[0] * last.shape[2]) < 4 * UNIT["float16"]


def test_two_streams_at_once(built):
    import torch
    import tf_approximate_b200 as ax
    cases = [make(s, "bfloat16", "float32") + (g,) for s, g in (((64, 28, 28, 64), 16), ((2, 160, 160, 128), 32), ((31, 27, 45, 120), 24))]
    def run(x, scale, offset, residual, grad, groups):
        y, st = ax.group_norm_forward(x, groups, scale, offset, residual, "silu")
        return (y, *ax.group_norm_backward(grad, x, st, groups, scale, offset, residual, "silu"))
    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(4):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(run(*c))
    torch.cuda.synchronize()
    for w, all_ in zip(want, got):
        for g in all_:
            assert all(torch.equal(a, b) for a, b in zip(w, g))


def test_refusals(built):
    import torch
    import tf_approximate_b200 as ax
    x = torch.randn(2, 4, 8, device="cuda")
    s = torch.ones(8, device="cuda")
    y, statistics = ax.group_norm_forward(x, 2)
    for call in (lambda: ax.group_norm(x, 3), lambda: ax.group_norm(x, 0), lambda: ax.group_norm(x, -1), lambda: ax.group_norm(x.double(), 2), lambda: ax.group_norm(x[0, 0], 2),
                 lambda: ax.group_norm(x, 2, s[:4]), lambda: ax.group_norm(x, 2, s.double()), lambda: ax.group_norm(x, 2, s.cpu()), lambda: ax.group_norm(x, 2, s, s, x[:1]),
                 lambda: ax.group_norm(x, 2, residual=x.half()), lambda: ax.group_norm(x, 2, epsilon=-1.0), lambda: ax.group_norm(x, 2, epsilon=float("nan")),
                 lambda: ax.group_norm(x, 2, activation="tanh"), lambda: ax.group_norm(x.cpu(), 2), lambda: ax.group_norm(torch.zeros(2, 0, device="cuda"), 1),
                 lambda: ax.group_norm_backward(x, x, statistics, 4), lambda: ax.group_norm_backward(x[:1], x, statistics, 2), lambda: ax.group_norm_backward(x, x, y, 2),
                 lambda: ax.group_norm_backward(x, x, statistics.double(), 2), lambda: ax.GroupNorm(10, 4), lambda: ax.GroupNorm(8, 2, activation="tanh")):
        with pytest.raises(ax.InvalidArgumentError):
            call()
