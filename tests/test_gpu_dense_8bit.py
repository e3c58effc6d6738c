"""GPU: block quantisation to the bit of its definition, and the dense layer on 8-bit operands against 64 bits.

Bounds.  Codes and scales are exact, so the sums are compared with those of the quantised operands.  Of S = |x| |kernel|: the matrix pipes cut a sum off
at 2^-23 of it at each step of 32 inputs, or of 16, so at most 8 times within a block of 128, whose product with its scale is rounded
to fp32 and added to the others: (8 + 1) 2^-23 S in all for the blocks' own sums, 2^-24 S for each addition of a block.  Bias and residual make two more
additions, y is rounded once.  The activations' slopes are below 1.13, their own errors below 2^-20 of their argument (2^-17 for 16-bit results)."""
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-44, "bfloat16": 1e-40, "float16": 2.0 ** -25}
SIZES = [(1, 1, 1), (1, 128, 16), (1, 4096, 1000), (2, 129, 17), (3, 127, 33), (8, 300, 200), (8, 8000, 40), (8, 9000, 40), (9, 128, 128), (1, 70000, 20), (16, 1030, 77), (33, 16, 300), (127, 640, 129),
         (129, 641, 127), (256, 2048, 1000), (300, 1030, 500), (640, 24, 5000), (1531, 130, 277)]


def exact_quantized(x, rows):
    """Codes' values and scales by the definition, in 64 bits."""
    import torch
    r, k = x.shape
    d = torch.nn.functional.pad(x.double(), (0, -k % 128, 0, -r % rows)).view(-(-r // rows), rows, -(-k // 128), 128)
    top = d.abs().amax((1, 3)).clamp(min=2.0 ** -126)
    part, power = torch.frexp(top)                       # part in [1/2, 1): 448 is 7/8 of 2^9
    scale = torch.ldexp(torch.ones_like(part), (power - 9 + (part > 0.875).int()).clamp(min=-126))
    v = d / scale[:, None, :, None]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    v = torch.round(v / step) * step                     # to even
    return v.reshape(-(-r // rows) * rows, -1)[:r, :k], scale


def spread(values, scales, rows):
    """Quantised operands as they stand, in 64 bits."""
    r, k = values.shape
    return values.double() * scales.double().repeat_interleave(rows, 0)[:r].repeat_interleave(128, 1)[:, :k]


def make(r, k, u, dtype, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + r + k + u)
    dt = getattr(torch, dtype)
    x = torch.randn(r, k, device="cuda", generator=g) * torch.exp(torch.randn(r, 1, device="cuda", generator=g))
    w = torch.randn(u, k, device="cuda", generator=g) * k ** -0.5
    return x.to(dt), w, torch.randn(u, device="cuda", generator=g).to(dt), torch.randn(r, u, device="cuda", generator=g).to(dt), g


def check_dense8(x, codes, scales, bias=None, residual=None, act=None):
    import torch
    import tf_approximate_b200 as ax
    F = torch.nn.functional
    dtype = str(x.dtype)[6:]
    y = ax.dense_8bit(x, codes, scales, bias, residual, act, check=True)
    assert y.dtype == x.dtype and y.shape == (*x.shape[:-1], codes.shape[0]) and y.is_contiguous()
    rows = x.reshape(-1, x.shape[-1])
    a, w = spread(*exact_quantized(rows, 1), 1), spread(codes, scales, 128)
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    b, res = zero if bias is None else bias.double(), zero if residual is None else residual.reshape(-1, codes.shape[0]).double()
    z = a @ w.t() + b + res
    blocks = -(-x.shape[-1] // 128)
    off = (a.abs() @ w.abs().t()) * (9 * 2.0 ** -23 + blocks * 2.0 ** -24) + 3 * 2.0 ** -24 * (z.abs() + b.abs() + res.abs())
    want = {None: lambda v: v, "relu": torch.relu, "gelu": F.gelu, "silu": F.silu}[act](z)
    own = (2.0 ** -20 if dtype == "float32" else 2.0 ** -17) * z.abs() if act in ("gelu", "silu") else 0.0
    assert bool(((y.reshape(-1, codes.shape[0]).double() - want).abs() <= 1.13 * off + own + UNIT[dtype] * want.abs() + TINY[dtype]).all())
    return y


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("r,k", [(1, 1), (1, 128), (3, 129), (5, 8), (128, 128), (129, 127), (260, 1030), (64, 4096)])
def test_codes_and_scales(built, r, k, dtype):
    import torch
    import tf_approximate_b200 as ax
    x, _, _, _, g = make(r, k, 1, dtype)
    x[r // 2] *= 0                                      # a row of zeros
    for rows in (1, 128):
        codes, scales = ax.quantize_blocks(x, rows)
        want, want_scales = exact_quantized(x, rows)
        assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape and torch.equal(scales.double(), want_scales) and torch.equal(codes.double(), want)


def test_codes_at_the_edges(built):
    """Ties, the largest code, values that no scale brings into range, and blocks that have none."""
    import torch
    import tf_approximate_b200 as ax
    x = torch.zeros(8, 256, device="cuda")
    x[0, :6] = torch.tensor([448.0, 17.0, 19.0, -17.0, 2.0 ** -10, 3 * 2.0 ** -10])       # ties to even, between codes and below the smallest
    x[1, 0], x[2, 0], x[3, 0] = 448.0 + 2.0 ** -15, 1.75 * 2.0 ** 100, 3.0e38
    x[4, :2] = torch.tensor([2.0 ** -126, -(2.0 ** -149)])
    codes, scales = ax.quantize_blocks(x)
    want, want_scales = exact_quantized(x, 1)
    assert torch.equal(codes.double(), want) and torch.equal(scales.double(), want_scales)
    x[5, 3], x[6, 130] = float("inf"), float("nan")
    codes, scales = ax.quantize_blocks(x)
    bad = torch.zeros(8, 2, dtype=torch.bool, device="cuda")
    bad[5, 0] = bad[6, 1] = True
    assert torch.equal(scales.isnan(), bad)
    kernel, ks = ax.quantize_blocks(torch.randn(40, 256, device="cuda"), 128)
    for rows in (slice(0, 8), slice(None)):              # both kernels
        z = x[rows] if rows.stop else torch.cat([x] * 3)
        y = ax.dense_8bit(z, kernel, ks)
        bad_rows = ~z.isfinite().all(1)
        assert bool(y[bad_rows].isnan().all()) and bool(y[~bad_rows][0].isfinite().all())
    assert bool((ax.dense_8bit(torch.zeros(9, 256, device="cuda"), kernel, ks) == 0).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("r,k,u", SIZES)
def test_sizes(built, r, k, u, dtype):
    import tf_approximate_b200 as ax
    x, w, b, res, _ = make(r, k, u, dtype)
    codes, scales = ax.quantize_blocks(w, 128)
    n = r + k + u
    check_dense8(x, codes, scales, b if n % 2 else None, res if n % 3 else None, (None, "relu", "gelu", "silu")[n % 4])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
def test_activations_with_every_addition(built, act, dtype):
    import tf_approximate_b200 as ax
    for r in (5, 70):
        x, w, b, res, _ = make(r, 200, 150, dtype, 3)
        codes, scales = ax.quantize_blocks(w, 128)
        for bias in (b, b.float(), None):
            for residual in (res, None):
                check_dense8(x, codes, scales, bias, residual, act)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_tiles_and_split_sums(built, dtype):
    import tf_approximate_b200 as ax
    for r, k, u in ((2100, 136, 4500), (300, 16400, 200), (5000, 40, 264), (700, 1500, 700)):
        x, w, b, _, _ = make(r, k, u, dtype, 9)
        check_dense8(x, *ax.quantize_blocks(w, 128), b, None, "silu")


def test_strides_and_alignment(built):
    import torch
    import tf_approximate_b200 as ax
    for r in (4, 60):
        x, w, b, res, g = make(r, 272, 100, "bfloat16")
        codes, scales = ax.quantize_blocks(w, 128)
        raw = codes.view(torch.uint8)
        def placed(offset, line):
            room = torch.zeros(100 * line + offset, dtype=torch.uint8, device="cuda")
            v = room[offset:].view(100, line)[:, :272]
            v.copy_(raw)
            return v.view(torch.float8_e4m3fn)
        kernels = [codes, placed(0, 288), placed(1, 272), placed(16, 300), placed(8, 304), raw.t().contiguous().t().view(torch.float8_e4m3fn)]
        def rows(wide, from_, step=1):
            v = torch.zeros(r, wide, dtype=x.dtype, device="cuda")[:, from_::step][:, :272]
            v.copy_(x)
            return v
        xs = [x, rows(300, 5), rows(288, 8), x.t().contiguous().t(), rows(600, 0, 2), x[:1].expand(r, 272)]
        ss = [scales, scales.t().contiguous().t(), torch.stack([scales, scales], 2)[..., 0], scales, scales, scales]
        rs = [res, res.t().contiguous().t(), torch.cat([res, res], 1)[:, 3:103], res[:1].expand(r, 100), None, res]
        want = None
        for k, xi, s, re in zip(kernels, xs, ss, rs):
            check_dense8(xi, k, s, torch.stack([b, b], 1)[:, 0], re, "gelu")
            y = ax.dense_8bit(x, k, s)
            assert want is None or torch.equal(y, want)
            want = y
        assert torch.equal(ax.dense_8bit(x.view(2, r // 2, 272), codes, scales), want.view(2, r // 2, 100))
        q, qs = ax.quantize_blocks(rows(300, 5))
        assert torch.equal(q.view(torch.uint8), ax.quantize_blocks(x)[0].view(torch.uint8)) and torch.equal(qs, ax.quantize_blocks(x)[1])


def test_rows_do_not_depend_on_one_another(built):
    """A row of a call is the same whatever the other rows are (the same kernel taken), and the same every time."""
    import torch
    import tf_approximate_b200 as ax
    for r in (7, 300):
        x, w, b, _, _ = make(r, 1030, 333, "float16")
        codes, scales = ax.quantize_blocks(w, 128)
        y = ax.dense_8bit(x, codes, scales, b)
        z = x.clone()
        z[1:] = 7.0
        assert torch.equal(y[0], ax.dense_8bit(z, codes, scales, b)[0]) and torch.equal(y, ax.dense_8bit(x, codes, scales, b))


def test_scales_of_any_size(built):
    """fp32 scales that are no powers of two, far apart, and some whose product with a row's leaves fp32's range over a block of zeros."""
    import torch
    import tf_approximate_b200 as ax
    for r in (3, 40):
        x, w, _, _, g = make(r, 384, 200, "float32")
        codes, scales = ax.quantize_blocks(w, 128)
        scales = scales * (0.1 + torch.rand(scales.shape, device="cuda", generator=g) * 1e3)
        check_dense8(x, codes, scales)
        codes.view(torch.uint8)[:, 128:256] = 0
        scales[:, 1] = 3e38
        x[:, 128:256] *= 1e30
        check_dense8(x, codes, scales)


def test_empty_and_layer(built):
    import torch
    import tf_approximate_b200 as ax
    codes, scales = ax.quantize_blocks(torch.randn(40, 50, device="cuda"), 128)
    assert ax.dense_8bit(torch.zeros(0, 50, device="cuda"), codes, scales).shape == (0, 40)
    assert ax.dense_8bit(torch.zeros(3, 50, device="cuda"), codes[:0], scales[:0]).shape == (3, 0)
    assert ax.quantize_blocks(torch.zeros(0, 50, device="cuda"))[1].shape == (0, 1)
    torch.manual_seed(1)
    dense = ax.Dense(1030, 77, activation="silu").cuda()
    with torch.no_grad():
        dense.bias.normal_()
    layer = ax.Dense8bit(dense)
    assert not list(layer.parameters()) and layer.kernel.shape == (77, 1030) and layer.kernel.stride(0) % 16 == 0
    x = torch.randn(4, 6, 1030, device="cuda", requires_grad=True)
    y = layer(x)
    assert torch.equal(y, check_dense8(x.detach(), layer.kernel, layer.scales, layer.bias, None, "silu"))
    # an answer in 8 bits: 1024 products, each of two operands off by 2^-4 of themselves at most, by 2^-5 on average
    with torch.no_grad():
        assert float((y - dense(x)).norm() / dense(x).norm()) < 0.06
    again = ax.Dense8bit(ax.Dense(1030, 77, activation="silu").cuda())
    again.load_state_dict(layer.state_dict())
    assert torch.equal(again(x), y)


def test_captured_with_another_call_beside_it(built):
    import torch
    import tf_approximate_b200 as ax
    x, w, b, _, _ = make(200, 600, 333, "bfloat16")
    codes, scales = ax.quantize_blocks(w, 128)
    first, few = ax.dense_8bit(x, codes, scales, b, None, "gelu"), ax.dense_8bit(x[:2], codes, scales, b, None, "gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = ax.dense_8bit(x, codes, scales, b, None, "gelu"), ax.dense_8bit(x[:2], codes, scales, b, None, "gelu")
            graphs.append((g, out))
    torch.cuda.current_stream().wait_stream(side)
    for g, out in graphs + graphs:
        g.replay()
        assert torch.equal(ax.dense_8bit(x, codes, scales, b, None, "gelu"), first)
        torch.cuda.synchronize()
        assert torch.equal(out[0], first) and torch.equal(out[1], few)


def test_a_kernel_of_more_bytes_than_31_bits_count(built):
    """70016 units of 32768 inputs: the last units' answers, for few rows and for many."""
    import torch
    import tf_approximate_b200 as ax
    g = torch.Generator(device="cuda").manual_seed(2)
    units, inputs = 70016, 32768
    codes = torch.randint(0, 0x7f, (units, inputs), dtype=torch.uint8, device="cuda", generator=g).view(torch.float8_e4m3fn)      # any code but NaN
    scales = torch.full((units // 128, inputs // 128), 2.0 ** -12, device="cuda")
    for r in (2, 40):
        x = torch.randn(r, inputs, device="cuda", generator=g)
        y = ax.dense_8bit(x, codes, scales, check=True)
        a, w = spread(*exact_quantized(x, 1), 1), codes[-200:].double() * 2.0 ** -12
        # as above: 9 2^-23 for the blocks' own sums, 2^-24 for each of 256 additions
        assert bool(((y[:, -200:].double() - a @ w.t()).abs() <= (a.abs() @ w.abs().t()) * (9 * 2.0 ** -23 + 256 * 2.0 ** -24)).all())


def test_two_streams_at_once(built):
    import torch
    import tf_approximate_b200 as ax
    cases = [make(r, k, u, "bfloat16")[:3] for r, k, u in ((3, 4096, 3000), (200, 1030, 777), (1500, 512, 2000))]
    operands = [(x, *ax.quantize_blocks(w, 128), b) for x, w, b in cases]
    want = [ax.dense_8bit(*o) for o in operands]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in operands], []
    for _ in range(5):
        for i, (o, s) in enumerate(zip(operands, streams)):
            with torch.cuda.stream(s):
                got.append((i, ax.dense_8bit(*o)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)


def test_refusals(built):
    import torch
    import tf_approximate_b200 as ax
    x, w = torch.randn(4, 200, device="cuda"), torch.randn(300, 200, device="cuda")
    c, s = ax.quantize_blocks(w, 128)
    b = torch.zeros(300, device="cuda")
    grad = x.clone().requires_grad_()
    for call in (lambda: ax.dense_8bit(x.double(), c, s), lambda: ax.dense_8bit(x, w, s), lambda: ax.dense_8bit(x, c.view(torch.uint8), s), lambda: ax.dense_8bit(x[:, :100], c, s),
                 lambda: ax.dense_8bit(x, c, s[:2]), lambda: ax.dense_8bit(x, c, s.half()), lambda: ax.dense_8bit(x, c, s[:, :1]), lambda: ax.dense_8bit(x, c, s.cpu()), lambda: ax.dense_8bit(x, c, s, b[:5]),
                 lambda: ax.dense_8bit(x, c, s, b.double()), lambda: ax.dense_8bit(x, c, s, b, x), lambda: ax.dense_8bit(x, c, s, activation="tanh"), lambda: ax.dense_8bit(x.cpu(), c, s),
                 lambda: ax.dense_8bit(grad, c, s), lambda: ax.dense_8bit(x, c, s, b.requires_grad_()), lambda: ax.quantize_blocks(x, 2), lambda: ax.quantize_blocks(x.double()),
                 lambda: ax.quantize_blocks(x.view(2, 2, 200), 128), lambda: ax.quantize_blocks(x.cpu()), lambda: ax.Dense8bit(torch.nn.Linear(3, 4))):
        with pytest.raises(ax.InvalidArgumentError):
            call()
