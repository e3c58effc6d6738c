"""GPU: the AdamW step against its formula in 64 bits, step by step from the state the kernel itself has, and its refusals."""
import math

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                       # half a unit in the last place of fp32, relative
TYPE_U = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
# sizes at the edges of the blocks of 256 values, of a warp's and a CTA's work, and one of nothing
SIZES = [1, 255, 256, 257, 3, 0, 2048, 2049, 7, 8192 * 3 + 5, 40000]


def _moments(opt):
    if opt.state_bits == 32:
        return opt.exp_avg.double(), opt.exp_avg_sq.double()
    m = (opt.exp_avg.double().view(-1, 256) * opt.exp_avg_scale.double()[:, None]).view(-1)
    r = (opt.exp_avg_sq_root.double().view(-1, 256) * opt.exp_avg_sq_root_scale.double()[:, None]).view(-1)
    return m, r * r


def _near_codes(values, codes, scale, root):
    """Every code is the nearest to its value of those that a scale of this block has (one rounding of the scale, one of the quotient)."""
    import torch
    v, q = values.view(-1, 256), codes.double().view(-1, 256)
    top = v.abs().amax(1)
    assert torch.allclose(scale.double() * 448.0, top, rtol=8 * U, atol=0)
    s = scale.double()[:, None]
    half = torch.maximum(v.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -10)
    if root:
        half = torch.where((v > 0) & (v < s * 2.0 ** -9), s * 2.0 ** -9, half)
        assert bool((q[v > s * 1e-30] > 0).all())
    assert bool(((q * s - v).abs() <= half).all())


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_steps_follow_the_formula(built, dtype, bits, offset):
    import torch
    import tf_approximate_b200 as ax
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(bits + offset)
    params = [(torch.randn(n + offset, device="cuda", generator=g) * 0.1).to(dt)[offset:] for n in SIZES]     # also off the 16-byte grid
    lr, betas, eps, decay, scale = 1e-2, (0.9, 0.999), 1e-8, 0.1, 0.25
    opt = ax.AdamW([{"params": params[:4]}, {"params": params[4:], "lr": 3 * lr, "weight_decay": 0.0}], lr, betas, eps, decay, bits)
    starts, at = [], 0
    for n in SIZES:
        starts.append(at)
        at += -(-n // 256) * 256
    for step in range(1, 4):
        grads = [(torch.randn(n + offset, device="cuda", generator=g) * 10.0 ** (step - 3)).to(dt)[offset:] for n in SIZES]
        for k in (0, 3):
            grads[k][:1] = 0
        before, (m0, v0) = [p.double() for p in params], _moments(opt)
        opt.step(grads, grad_scale=scale)
        m1, v1 = _moments(opt)
        want_m, want_v = torch.zeros_like(m0), torch.zeros_like(v0)
        for i, n in enumerate(SIZES):
            at = slice(starts[i], starts[i] + n)
            gi = grads[i].double() * scale
            m = m0[at] * betas[0] + gi * (1 - betas[0])
            v = v0[at] * betas[1] + gi * gi * (1 - betas[1])
            want_m[at], want_v[at] = m, v
            rate, wd = (lr, decay) if i < 4 else (3 * lr, 0.0)
            move = rate / (1 - betas[0] ** step) * m / (v.sqrt() / math.sqrt(1 - betas[1] ** step) + eps)
            want = before[i] * (1 - rate * wd) - move
            # m: two roundings of values up to |m0| + |g|; the quotient: those, relative to the denominator, and some 2^-21 of its own
            off_m = 4 * U * (m0[at].abs() + gi.abs())
            den = v.sqrt() / math.sqrt(1 - betas[1] ** step) + eps
            off = rate / (1 - betas[0] ** step) * off_m / den + 32 * U * move.abs() + 4 * U * before[i].abs() + TYPE_U[dtype] * want.abs()
            off = off * 1.01 + (2.0 ** -25 if dtype == "float16" else 0.0)
            assert bool(((params[i].double() - want).abs() <= off).all()), (i, step)
        if bits == 32:
            assert bool(((m1 - want_m).abs() <= 4 * U * (m0.abs() + 10 * want_m.abs() + 9 * m0.abs())).all())
            assert bool(((v1 - want_v).abs() <= 8 * U * (v0 + want_v)).all())
        else:
            _near_codes(want_m, opt.exp_avg, opt.exp_avg_scale, False)
            _near_codes(want_v.sqrt(), opt.exp_avg_sq_root, opt.exp_avg_sq_root_scale, True)
    assert opt.step_count == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_table(built, bits):
    """1000 tensors take two launches of the large table; each moves by lr against the sign of its gradient in the first step."""
    import torch
    import tf_approximate_b200 as ax
    params = [torch.zeros(1 + i % 300, device="cuda") for i in range(1000)]
    grads = [torch.full_like(p, 1.0 if i % 2 else -1.0) for i, p in enumerate(params)]
    opt = ax.AdamW(params, lr=0.5, weight_decay=0.0, state_bits=bits)
    opt.step(grads)
    for i, p in enumerate(params):
        assert torch.allclose(p, torch.full_like(p, -0.5 if i % 2 else 0.5), rtol=1e-6), i


@pytest.mark.parametrize("missing", [(0,), (1, 2), (4,), (0, 1, 2, 3, 4)])
def test_parameters_without_gradient_stay(built, missing):
    import torch
    import tf_approximate_b200 as ax
    params = [torch.full((n,), 2.0, device="cuda") for n in (5, 300, 256, 1000, 9)]
    opt = ax.AdamW(params, lr=0.25, weight_decay=0.0, state_bits=8)
    for i, p in enumerate(params):
        p.grad = None if i in missing else torch.ones_like(p)
    opt.step()
    for i, p in enumerate(params):
        assert torch.allclose(p, torch.full_like(p, 2.0 if i in missing else 1.75), rtol=1e-6)
    at = 0
    for i, p in enumerate(params):
        n = -(-p.numel() // 256)
        assert bool((opt.exp_avg_scale[at:at + n] > 0).any()) == (i not in missing)
        at += n
    opt.zero_grad()
    assert all(p.grad is None for p in params)


def test_gradients_that_are_not_finite(built):
    """An infinity or a NaN stays in its own block of moments and its own parameter."""
    import torch
    import tf_approximate_b200 as ax
    for bits in (32, 8):
        p = torch.ones(1024, device="cuda")
        g = torch.ones(1024, device="cuda")
        g[300], g[900] = float("nan"), float("inf")
        opt = ax.AdamW([p], lr=0.5, weight_decay=0.0, state_bits=bits)
        opt.step([g])
        bad = ~torch.isfinite(p)
        assert bad.nonzero()[:, 0].tolist() in ([300, 900], [300])
        assert torch.allclose(p[:256], torch.full_like(p[:256], 0.5))
        m = opt.exp_avg.float()
        assert bool(torch.isfinite(m[:256]).all()) and bool(torch.isfinite(m[512:768]).all())


def test_gradients_with_strides_streams_and_state(built):
    import torch
    import tf_approximate_b200 as ax
    g = torch.Generator(device="cuda").manual_seed(3)
    a = [torch.randn(40, 30, device="cuda", generator=g), torch.randn(77, device="cuda", generator=g)]
    b = [t.clone() for t in a]
    grads = [torch.randn(30, 40, device="cuda", generator=g).t(), torch.randn(154, device="cuda", generator=g)[::2]]
    one, two = ax.AdamW(a, state_bits=8), ax.AdamW(b, state_bits=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for step in range(2):
        one.step(grads)
        with torch.cuda.stream(side):
            two.step([t.contiguous() for t in grads])
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    three = ax.AdamW(b, state_bits=8)
    three.load_state_dict(one.state_dict())
    one.step(grads)
    three.step(grads)
    assert three.step_count == 3 and all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals(built):
    import torch
    import tf_approximate_b200 as ax
    p = torch.zeros(4, 6, device="cuda")
    for bad in ([], [p, p], [p, p.clone().half()], [torch.zeros(3)], [p.t()], [p.double()]):
        with pytest.raises(ax.InvalidArgumentError):
            ax.AdamW(bad)
    for options in ({"state_bits": 16}, {"betas": (1.0, 0.9)}, {"eps": -1.0}):
        with pytest.raises(ax.InvalidArgumentError):
            ax.AdamW([p], **options)
    opt = ax.AdamW([p])
    for grads in ([], [torch.zeros(5, device="cuda")], [torch.zeros(4, 6)], [torch.zeros(4, 6, device="cuda").half()]):
        with pytest.raises(ax.InvalidArgumentError):
            opt.step(grads)
    opt.params.append(p.clone())
    with pytest.raises(ax.InvalidArgumentError):
        opt.step([p, p])
    opt.params.pop()
    assert opt.step_count == 0
    with pytest.raises(ax.InvalidArgumentError):
        opt.load_state_dict(ax.AdamW([p], state_bits=8).state_dict())
