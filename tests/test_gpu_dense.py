"""GPU: the exact dense layer and its gradients against 64 bits, at the edges of the tiles, types, layouts and strides, and its refusals.

Bounds.  S = |x| |kernel| + |bias| + |residual| bounds every partial sum.  16-bit operands: the tensor cores cut a sum off at 2^-23 of it
at each step of 16 products, and y is rounded once.  fp32 operands: the products of terms that are left out are below 2^-25 S, the sums
of 64 products lose at most 6 2^-23 S, and there is one fp32 addition for each 64.  The slopes of the activations are below 1.13, their
second derivatives below 0.8."""
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-44, "bfloat16": 1e-40, "float16": 2.0 ** -25}
SIZES = [(1, 1, 1), (1, 64, 128), (1, 520, 1000), (2, 63, 10), (16, 8, 257), (17, 129, 64), (33, 256, 130), (128, 64, 128), (129, 65, 127),
         (256, 2048, 1000), (300, 7, 520), (1000, 72, 33), (513, 320, 769)]


def sum_error(k, dtype):
    return (8 + k / 128) * 2.0 ** -23 if dtype == "float32" else (k / 16 + 4) * 2.0 ** -23


def exact_activation(z, name):
    import torch
    F = torch.nn.functional
    return {None: lambda v: v, "relu": torch.relu, "gelu": F.gelu, "silu": F.silu}[name](z)


def make(t, k, n, dtype, order, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + t + k + n)
    dt = getattr(torch, dtype)
    x = torch.randn(t, k, device="cuda", generator=g).to(dt)
    w = torch.randn((k, n) if order == "in_out" else (n, k), device="cuda", generator=g).to(dt)
    return x, w if order == "in_out" else w.t(), torch.randn(n, device="cuda", generator=g).to(dt), torch.randn(t, n, device="cuda", generator=g).to(dt), g


def check_dense(x, w, b, r, act, dtype, grad):
    import torch
    import tf_approximate_b200 as ax
    u, tiny = UNIT[dtype], TINY[dtype]
    y, kept = ax.dense_forward(x, w, b, r, act, check=True)
    assert y.dtype == x.dtype and y.is_contiguous()
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    xd, wd, bd, rd = [zero if v is None else v.double() for v in (x, w, b, r)]
    z = xd @ wd + bd + rd
    size = xd.abs() @ wd.abs() + bd.abs() + rd.abs()
    k, (t, n) = x.shape[-1], z.shape
    off_z = size * sum_error(k, dtype)
    want = exact_activation(z, act)
    assert bool(((y.double() - want).abs() <= 1.13 * off_z + want.abs() * (u + 2.0 ** -20) + tiny).all())
    dx, dw, db, dr = ax.dense_backward(grad, x, w, kept, act, bias=b, residual=r, check=True)
    gd = grad.double()
    if act == "relu":
        slope, off_slope = (y > 0).double(), torch.zeros_like(z)      # where z is within its error of zero, either slope is one
    else:
        zz = z.detach().requires_grad_()
        slope, = torch.autograd.grad(exact_activation(zz, act).sum(), zz) if act else (torch.ones_like(z),)
        off_slope = (0.8 * (off_z + u * z.abs() + tiny) + 2.0 ** -20) if act else torch.zeros_like(z)
    dz = gd * slope
    off_dz = gd.abs() * off_slope + (u * dz.abs() + tiny if act and dtype != "float32" else 2.0 ** -24 * dz.abs())
    for got, want, s, off, depth in ((dx, dz @ wd.t(), dz.abs() @ wd.t().abs(), off_dz @ wd.t().abs(), n),
                                     (dw, xd.t() @ dz, xd.t().abs() @ dz.abs(), xd.t().abs() @ off_dz, t)):
        assert got.shape == want.shape
        assert bool(((got.double() - want).abs() <= 1.01 * off + s * sum_error(depth, dtype) + want.abs() * u + tiny).all())
    if b is not None:
        assert bool(((db.double() - dz.sum(0)).abs() <= 1.01 * (gd.abs() * off_slope).sum(0) + (t + 8) * 2.0 ** -24 * dz.abs().sum(0)
                     + UNIT[str(b.dtype)[6:]] * dz.sum(0).abs() + TINY[str(b.dtype)[6:]]).all())
    if r is not None:
        assert dr.shape == r.shape and bool(((dr.double() - dz).abs() <= 1.01 * (gd.abs() * off_slope) + u * dz.abs() + tiny).all())
    assert (dw.stride(0) == 1) == (w.stride(0) == 1) or 1 in dw.shape


@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("t,k,n", SIZES)
def test_sizes(built, t, k, n, dtype, order):
    x, w, b, r, g = make(t, k, n, dtype, order)
    import torch
    grad = torch.randn(t, n, device="cuda", generator=g).to(x.dtype)
    check_dense(x, w, b, r if (t + n) % 2 else None, ("relu", "gelu", "silu", None)[(t + k + n) % 4], dtype, grad)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
def test_activations_with_every_addition(built, act, dtype):
    import torch
    for bias in (False, True):
        for residual in (False, True):
            x, w, b, r, g = make(70, 96, 200, dtype, "in_out", 5)
            grad = torch.randn(70, 200, device="cuda", generator=g).to(x.dtype)
            check_dense(x, w, b if bias else None, r if residual else None, act, dtype, grad)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_many_tiles_and_split_sums(built, dtype):
    """More tiles than SMs of either kind of tile, and a long k with few tiles."""
    import torch
    for t, k, n in ((2100, 136, 4500), (300, 16400, 200), (9000, 40, 264)):
        x, w, b, r, g = make(t, k, n, dtype, "out_in", 9)
        check_dense(x, w, b, None, "silu", dtype, torch.randn(t, n, device="cuda", generator=g).to(x.dtype))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides_and_alignment(built, dtype):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(dt)
    t, k, n = 130, 72, 136
    grad = rand(t, n)
    xs = [rand(k, t).t(), rand(t, k + 5)[:, 3:3 + k], rand(t, 2 * k)[:, ::2], rand(2 * t, k)[::2], rand(1, k).expand(t, k), rand(t * k + 1)[1:].view(t, k)]
    ws = [rand(k, n + 8)[:, 8:], rand(k, n + 1)[:, 1:], rand(n, k + 3)[:, :k].t(), rand(2 * k, n)[::2], rand(k, 1).expand(k, n), rand(k, 2 * n)[:, ::2]]
    rs = [rand(t, n + 4)[:, 4:], rand(n, t).t(), rand(1, n).expand(t, n), None, rand(2 * t, n)[::2], rand(t * n + 1)[1:].view(t, n)]
    for x, w, r in zip(xs, ws, rs):
        check_dense(x, w, rand(2 * n)[::2], r, "gelu", dtype, grad)
        check_dense(x, w, rand(n), r, None, dtype, rand(n, t).t())


@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9])
def test_few_rows(built, rows, dtype, order):
    """The kernels for up to 8 rows: short and long inputs, few units and many, off the 16-byte grid."""
    import torch
    for k, n in ((1, 5), (31, 260), (2048, 1000), (4100, 9999), (8192, 72), (264, 19000)):
        x, w, b, r, g = make(rows, k, n, dtype, order, 3)
        grad = torch.randn(rows, n, device="cuda", generator=g).to(x.dtype)
        check_dense(x, w, b, r, "silu" if k % 2 else None, dtype, grad)
    big = torch.randn(2 * rows, 301, device="cuda", generator=g).to(x.dtype)
    x, w, b, r, _ = make(rows, 300, 500, dtype, order, 4)
    check_dense(big[::2, 1:], w[:, 1:], b[1:], None, "gelu", dtype, r[:, 1:])


def test_bias_of_another_type_and_leading_dimensions(built):
    import torch
    import tf_approximate_b200 as ax
    x, w, b, r, g = make(24, 40, 56, "bfloat16", "in_out")
    y = ax.dense(x.view(2, 3, 4, 40), w, b.float(), r.view(2, 3, 4, 56), "relu")
    assert y.shape == (2, 3, 4, 56) and torch.equal(y.view(24, 56), ax.dense(x, w, b, r, "relu"))
    dx, dw, db, dr = ax.dense_backward(r.view(2, 3, 4, 56), x.view(2, 3, 4, 40), w, bias=b.float(), residual=y)
    assert dx.shape == (2, 3, 4, 40) and dw.shape == (40, 56) and db.dtype == torch.float32 and dr.shape == y.shape
    assert torch.equal(dx.view(24, 40), ax.dense_backward(r, x, w)[0])


def test_sizes_of_nothing(built):
    import torch
    import tf_approximate_b200 as ax
    for t, k, n in ((0, 8, 16), (5, 0, 16), (5, 8, 0), (0, 0, 0)):
        x, w, b = torch.ones(t, k, device="cuda"), torch.ones(k, n, device="cuda"), torch.full((n,), 2.0, device="cuda")
        y, kept = ax.dense_forward(x, w, b, None, "relu")
        assert y.shape == (t, n) and bool((y == 2).all() if k == 0 else True)
        dx, dw, db, _ = ax.dense_backward(torch.ones(t, n, device="cuda"), x, w, kept, "relu", bias=b)
        assert dx.shape == (t, k) and dw.shape == (k, n) and db.shape == (n,)
        assert bool((dx == 0).all()) and bool((dw == 0).all()) and bool((db == t).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_values_that_are_not_finite_stay_in_their_rows(built, dtype):
    import torch
    import tf_approximate_b200 as ax
    x, w, b, r, g = make(200, 100, 300, dtype, "in_out")
    clean = ax.dense(x, w)
    x[3, 5], x[150, 99] = float("inf"), float("nan")
    y = ax.dense(x, w)
    rows = torch.isfinite(y).all(1)
    assert (~rows).nonzero()[:, 0].tolist() == [3, 150]
    assert torch.equal(y[rows], clean[rows]) and not bool(torch.isfinite(y[[3, 150]]).any())
    if dtype == "float32":                      # beyond bf16's largest value, within fp32's
        big = torch.full((4, 64), 3.4e38, device="cuda")
        one = torch.zeros(64, 8, device="cuda")
        one[7] = 0.5
        assert torch.allclose(ax.dense(big, one), torch.full((4, 8), 1.7e38, device="cuda"), rtol=1e-6)


def test_streams_and_graphs(built):
    import torch
    import tf_approximate_b200 as ax
    x, w, b, r, g = make(300, 512, 700, "bfloat16", "out_in")
    want = ax.dense(x, w, b, r, "gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ax.dense(x, w, b, r, "gelu")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            replayed = ax.dense(x, w, b, r, "gelu")
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(replayed, want)


def test_autograd_of_the_layer(built):
    """Gradients through the layer are the explicit ones, and agree with differences of the output."""
    import torch
    import tf_approximate_b200 as ax
    torch.manual_seed(2)
    layer = ax.Dense(48, 40, activation="silu").cuda()
    x = torch.randn(30, 48, device="cuda", requires_grad=True)
    r = torch.randn(30, 40, device="cuda", requires_grad=True)
    g = torch.randn(30, 40, device="cuda")
    y = layer(x, r)
    y.backward(g)
    _, kept = ax.dense_forward(x, layer.kernel, layer.bias, r, "silu")
    explicit = ax.dense_backward(g, x, layer.kernel, kept, "silu", bias=layer.bias, residual=r)
    for p, e in zip((x, layer.kernel, layer.bias, r), explicit):
        assert torch.equal(p.grad, e)
    # along a direction: (f(p + h d) - f(p - h d)) / 2h; h = 2^-6: cut-off error h^2/6 |f'''| and 2^-22 of the sum of |g y| over h
    with torch.no_grad():
        for p in (x, layer.kernel, layer.bias, r):
            d = p.grad / p.grad.norm()
            h, f = 2.0 ** -6, []
            for sign in (1, -1):
                p += sign * h * d
                f.append((layer(x, r).double() * g.double()).sum())
                p -= sign * h * d
            slope = float((f[0] - f[1]) / (2 * h))
            assert abs(slope - float(p.grad.norm())) < 0.01 * float(p.grad.norm())
    with pytest.raises(RuntimeError):
        dx, = torch.autograd.grad(layer(x, r).sum(), x, create_graph=True)
        dx.sum().backward()


def test_refusals(built):
    import torch
    import tf_approximate_b200 as ax
    x, w, b, r, g = make(4, 8, 16, "float32", "in_out")
    for args in ((x.cpu(), w), (x, w.cpu()), (x.half(), w), (x.double(), w.double()), (x, w[:7]), (x, w[0]), (x, w, b[:3]), (x, w, b.double()), (x, w, b, r[:3]),
                 (x, w, b, r.half()), (x, w, b, r, "tanh"), (None, w)):
        with pytest.raises(ax.InvalidArgumentError):
            ax.dense(*args)
    for grad in (r[:2], r.half(), r.cpu()):
        with pytest.raises(ax.InvalidArgumentError):
            ax.dense_backward(grad, x, w)
    with pytest.raises(ax.InvalidArgumentError):
        ax.dense_backward(r, x, w, None, "gelu")
    with pytest.raises(ax.InvalidArgumentError):
        ax.Dense(4, 4, activation="tanh")
