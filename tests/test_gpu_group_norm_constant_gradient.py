"""GPU: group norm's dx where the gradient of its output is the same at all places, as behind a mean over them: dz is nearly the same all over a
group, next to nothing of it is left in dx, and any rounding of dz on the way would be most of that.

Bounds.  As in test_gpu_group_norm.py, with dx rounded once and nothing else to 16 bits.  D = 2^-24, K = 64: a group's mean is off by at most K D of its
largest value, r by K D of itself; z has four roundings on top; a slope's own error is below 2^-20 of 1 + |z| (2^-17 for 16-bit results), the second
derivatives are below 0.8; a sum is off by K D of its magnitudes and by what its terms are off; six roundings make dx of them."""
import pytest

pytestmark = pytest.mark.gpu

D, K = 2.0 ** -24, 64          # K: 1024 for the tensors that are read twice
UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-44, "bfloat16": 1e-40, "float16": 2.0 ** -25}
# spans of whole vectors, lines that start anywhere, a cluster, one block, tensors that are read twice
SHAPES = [((2, 16, 16, 64), 8), ((3, 9, 11, 20), 4), ((2, 40, 40, 256), 8), ((5, 27, 45, 120), 24), ((2, 160, 160, 128), 32), ((2, 40, 40, 2504), 1), ((1, 50, 40, 2500), 1)]


def check_dx(x, groups, scale, offset, residual, act, grad, k=K):
    import torch
    import tf_approximate_b200 as ax
    dtype, n, each = str(x.dtype)[6:], x.shape[0], x.shape[-1] // groups
    u, own, e = UNIT[dtype], 2.0 ** -20 if dtype == "float32" else 2.0 ** -17, k * D
    _, statistics = ax.group_norm_forward(x, groups, scale, offset, residual, act)
    dx, _, _, dr = ax.group_norm_backward(grad, x, statistics, groups, scale, offset, residual, act)
    def parts(t):
        return t.double().reshape(n, -1, groups, each)
    xd, gd, s, o = parts(x), parts(grad), scale.double().view(1, 1, groups, each), offset.double().view(1, 1, groups, each)
    var, mean = torch.var_mean(xd, (1, 3), correction=0, keepdim=True)
    r = 1 / torch.sqrt(var + 1e-3)
    xhat, add = (xd - mean) * r, parts(residual) if residual is not None else 0.0 * xd
    off_xhat = r * e * xd.abs().amax((1, 3), keepdim=True) + (e + 4 * D) * xhat.abs()
    z = (xhat * s + o + add).detach().requires_grad_()
    F = torch.nn.functional
    slope = torch.autograd.grad({"silu": F.silu, "gelu": F.gelu}[act](z).sum(), z)[0]
    z = z.detach()
    off_z = off_xhat * s.abs() + 4 * D * (z.abs() + o.abs() + add.abs())
    dz = gd * slope
    off_dz = gd.abs() * (0.8 * off_z + own * (1 + z.abs())) + 2 * D * dz.abs()
    m = xd.shape[1] * each
    m1, m2 = (dz * s).sum((1, 3), keepdim=True) / m, (dz * s * xhat).sum((1, 3), keepdim=True) / m
    off1 = ((off_dz + e * dz.abs()) * s.abs()).sum((1, 3), keepdim=True) / m
    off2 = ((off_dz * xhat.abs() + dz.abs() * (off_xhat + e * xhat.abs())) * s.abs()).sum((1, 3), keepdim=True) / m
    want = r * (dz * s - m1 - xhat * m2)
    off = r * (off_dz * s.abs() + off1 + xhat.abs() * off2 + off_xhat * m2.abs() + (e + 6 * D) * (dz.abs() * s.abs() + m1.abs() + xhat.abs() * m2.abs()))
    assert bool(((parts(dx) - want).abs() <= off + u * want.abs() + TINY[dtype]).all())
    if residual is not None:
        assert bool(((parts(dr) - dz).abs() <= off_dz + u * dz.abs() + TINY[dtype]).all())
    return float((parts(dx) - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("act,mean,dy", [("silu", 3.0, 1.0), ("silu", 6.0, 1.0), ("gelu", 4.0, 2.0 ** -11)])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_dx_is_rounded_once(built, shape, groups, act, mean, dy, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    dt, c = getattr(torch, dtype), shape[-1]
    def rand(*s):
        return torch.randn(*s, device="cuda", generator=g)
    x, scale, offset = rand(*shape).to(dt), (1 + 0.1 * rand(c)), mean + 0.1 * rand(c)
    grad = torch.full((), dy, device="cuda", dtype=dt).expand(shape)
    for residual in (None, (0.1 * rand(*shape)).to(dt)):
        check_dx(x, groups, scale, offset, residual, act, grad, 1024 if c > 2048 else K)
    # the same at addresses off 16 bytes: value by value
    if x.numel() < 1 << 16:
        for residual in (None, (0.1 * rand(*shape)).to(dt)):
            moved = torch.cat([x.flatten()[:1], x.flatten()])[1:].view(shape)
            check_dx(moved, groups, scale, offset, residual, act, grad)


def test_a_global_mean_behind_the_norm(built):
    """The gradient that autograd hands back from a mean over the places, in bf16."""
    import torch
    import tf_approximate_b200 as ax
    torch.manual_seed(5)
    x = torch.randn(4, 28, 28, 64, device="cuda").bfloat16().requires_grad_()
    layer = ax.GroupNorm(64, 8, activation="silu").cuda()
    with torch.no_grad():
        layer.offset.fill_(6.0)
    layer(x).mean((1, 2)).sum().backward()
    xd = x.detach().double().requires_grad_()
    y = torch.nn.functional.group_norm(xd.permute(0, 3, 1, 2), 8, layer.scale.detach().double(), layer.offset.detach().double(), 1e-3)
    # what the mean hands back in bf16
    grad = torch.full((), 1 / (28 * 28), device="cuda").bfloat16().double().expand(4, 28, 28, 64)
    torch.nn.functional.silu(y.permute(0, 2, 3, 1)).backward(grad)
    # a rounding to bf16 makes 0.0017 in all
    assert float((x.grad.double() - xd.grad).norm() / xd.grad.norm()) < 2.0 ** -8
