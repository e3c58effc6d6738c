"""What stands between and behind the table convolutions of a network, with the sizes that performance is measured at: group norm with
the shortcut and the activation that follow it, and its gradients (channels last); dropout whose mask is computed from a counter and
never stored; and the dense layer in 8-bit floating point, with a scale for each block of 128 values, that a trained network answers with.

A case is one pass through an operator.  With `own` false, `run` computes it in elementary torch operations in fp32, rounded once at the
end to the type of its output; with `own` true, by the calls of this package.  Sizes are those of the layers of the ResNet-50 and ResNet-20
workloads, and generic ones; `draw` gives more cases of the same ranges.

A ReLU is measured in forward passes: where its argument is within rounding of zero, either slope is as good as the other, and its gradient
tells nothing about either side."""
import math

import numpy as np
import torch

own = False

DEVICE = torch.device("cuda", 0)
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 128                # values that share a scale
EPSILON = 1e-3
LARGEST = 256 * 56 * 56 * 256


# ---------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------
def group_norm(samples, height, width, channels, groups, dtype, activation="none", residual=False, train=False, params="float32"):
    return {"op": "group_norm", "samples": samples, "height": height, "width": width, "channels": channels, "groups": groups, "dtype": dtype,
            "activation": activation, "residual": residual, "train": train, "params": params}


def dropout(rows, columns, rate, dtype, residual=False):
    return {"op": "dropout", "rows": rows, "columns": columns, "rate": rate, "dtype": dtype, "residual": residual}


def dense_8bit(rows, inputs, units, dtype, activation="none", bias=True, residual=False):
    return {"op": "dense_8bit", "rows": rows, "inputs": inputs, "units": units, "dtype": dtype, "activation": activation, "bias": bias,
            "residual": residual}


def listed():
    return [
        # one image in the last stage of ResNet-20, as a model answers it: a pass is latency
        dict(group_norm(1, 8, 8, 64, 8, "float32", "relu", residual=True), name="group_norm_one_image"),
        # a training step in the first stage of ResNet-20, in the type that the table convolutions work in; two channels a group
        dict(group_norm(1024, 32, 32, 16, 8, "float32", "silu", train=True), name="group_norm_resnet20"),
        # sizes that are multiples of nothing, five channels a group, a shortcut: a training step
        dict(group_norm(31, 27, 45, 120, 24, "float16", "gelu", residual=True, train=True, params="float16"), name="group_norm_ragged"),
        # few images with many places, as in segmentation: a group's values are more than any SM holds
        dict(group_norm(2, 512, 512, 128, 32, "bfloat16", "silu", train=True), name="group_norm_large_images"),
        # the widest tensor of ResNet-50 at the benchmark's batch, with its shortcut: a training step
        dict(group_norm(256, 56, 56, 256, 32, "bfloat16", "silu", residual=True, train=True), name="group_norm_resnet50"),
        # the features before the head of ResNet-50 at the benchmark's batch, and their gradient: a pass is latency
        dict(dropout(256, 2048, 0.2, "float32"), name="dropout_resnet50_head"),
        # a branch that is dropped before its shortcut is added, odd sizes
        dict(dropout(10007, 777, 0.35, "float16", residual=True), name="dropout_ragged"),
        # the widest tensor of ResNet-50 at the benchmark's batch
        dict(dropout(256 * 56 * 56, 256, 0.1, "bfloat16"), name="dropout_resnet50"),
        # one row through a wide layer, as a model answers one by one: the weights are read once, latency counts
        dict(dense_8bit(1, 4096, 16384, "bfloat16", "silu", bias=False), name="dense_8bit_one_row"),
        # the classifier of ResNet-50 at the benchmark's batch, in the type that the table convolutions work in
        dict(dense_8bit(256, 2048, 1000, "float32"), name="dense_8bit_resnet50_head"),
        # sizes that are multiples of nothing: blocks that end inside a line and inside a tile
        dict(dense_8bit(1531, 1030, 2777, "float16", "relu", residual=True), name="dense_8bit_ragged"),
        # the widening layer of a large block at a large batch: bound by the matrix units
        dict(dense_8bit(8192, 4096, 16384, "bfloat16", "gelu"), name="dense_8bit_large"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("group_norm", "group_norm", "dropout", "dense_8bit"))
    dtype = rng.choice(("bfloat16", "float16", "float32"))
    if op == "group_norm":
        groups, each = _log(rng, 1, 64), _log(rng, 1, 64)
        channels = groups * each
        samples, height, width = _log(rng, 1, 256), _log(rng, 1, 256), _log(rng, 1, 256)
        most = LARGEST // (2 if dtype == "float32" else 1)
        height = max(1, min(height, most // (width * channels)))
        # a group of a few values has a gradient that is nearly nothing but rounding
        height = max(height, -(-64 // (width * each)))
        samples = max(1, min(samples, most // (height * width * channels)))
        train = rng.random() < 0.7
        activation = rng.choice(("none", "gelu", "silu") if train else ("none", "relu", "gelu", "silu"))
        return group_norm(samples, height, width, channels, groups, dtype, activation, rng.random() < 0.4, train, rng.choice(("float32", dtype)))
    if op == "dropout":
        rows, columns = _log(rng, 1, 1 << 18), _log(rng, 16, 4096)
        rows = max(1, min(rows, LARGEST // 2 // columns))
        return dropout(rows, columns, rng.choice((0.05, 0.1, 0.25, 0.5, 0.9)), dtype, rng.random() < 0.4)
    rows, inputs, units = _log(rng, 1, 8192), _log(rng, 48, 4096), _log(rng, 40, 16384)
    return dense_8bit(rows, inputs, units, dtype, rng.choice(("none", "relu", "gelu", "silu")), rng.random() < 0.7, rng.random() < 0.4)


# ---------------------------------------------------------------------------------------------------
# what a user's program has in hand
# ---------------------------------------------------------------------------------------------------
def _normal(g, shape, scale, dtype):
    return (torch.randn(shape, device=DEVICE, generator=g) * scale).to(dtype)


def _blocks(x, rows):
    """x [r, k] in blocks of `rows` x 128, zeros behind its ends: [r / rows, rows, k / 128, 128]."""
    r, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -r % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // BLOCK, BLOCK)


def _quantize(x, rows):
    """e4m3 codes of x [r, k], and the scale of each block of `rows` x 128: the least power of two (2^-126 at least) with which the block's
    largest value is a code, 448 at most."""
    blocks = _blocks(x.float(), rows)
    part, power = torch.frexp(blocks.abs().amax((1, 3)).clamp(min=2.0 ** -126))
    power = (power - 9 + (part > 0.875).int()).clamp(min=-126)
    scales = torch.ldexp(torch.ones_like(part), power)
    codes = (blocks / scales[:, None, :, None]).to(torch.float8_e4m3fn)
    codes = codes.view(blocks.shape[0] * rows, -1)[:x.shape[0], :x.shape[1]].contiguous()
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    if case["op"] == "group_norm":
        shape, channels = (case["samples"], case["height"], case["width"], case["channels"]), case["channels"]
        # what a convolution hands over: channels of unequal size and with means of their own
        x = torch.randn(shape, device=DEVICE, generator=g)
        x = x.mul_(torch.exp(0.5 * torch.randn(channels, device=DEVICE, generator=g))).add_(torch.randn(channels, device=DEVICE, generator=g))
        return {"case": case, "x": x.to(dtype), "scale": (1.0 + _normal(g, (channels,), 0.2, torch.float32)).to(TYPES[case["params"]]),
                "offset": _normal(g, (channels,), 0.2, TYPES[case["params"]]),
                "residual": _normal(g, shape, 1.0, dtype) if case["residual"] else None,
                "grad": _normal(g, shape, 0.05, dtype) if case["train"] else None}
    if case["op"] == "dropout":
        shape = (case["rows"], case["columns"])
        return {"case": case, "x": _normal(g, shape, 1.0, dtype), "grad": _normal(g, shape, 0.05, dtype),
                "residual": _normal(g, shape, 1.0, dtype) if case["residual"] else None,
                "seed": (seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 63), "offset": seed % 1000}
    rows, inputs, units = case["rows"], case["inputs"], case["units"]
    # activations of very different size from row to row
    x = torch.randn((rows, inputs), device=DEVICE, generator=g) * torch.exp(torch.randn((rows, 1), device=DEVICE, generator=g))
    # the weights are quantised once, when a trained network is made ready to answer
    codes, scales = _quantize(_normal(g, (units, inputs), inputs ** -0.5, torch.float32), BLOCK)
    return {"case": case, "x": x.to(dtype), "codes": codes, "scales": scales, "bias": _normal(g, (units,), 0.1, dtype) if case["bias"] else None,
            "residual": _normal(g, (rows, units), 1.0, dtype) if case["residual"] else None}


# ---------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------
def _activate(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.7071067811865476))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * 0.7071067811865476)) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain_group_norm(state):
    case, x = state["case"], state["x"]
    out, shape = x.dtype, (case["samples"], case["height"] * case["width"], case["groups"], case["channels"] // case["groups"])
    x = x.float().view(shape)
    scale, offset = state["scale"].float().view(shape[2:]), state["offset"].float().view(shape[2:])
    count = shape[1] * shape[3]
    x = x - x.sum((1, 3), keepdim=True) / count
    root = torch.rsqrt((x * x).sum((1, 3), keepdim=True) / count + EPSILON)
    x = x * root
    z = x * scale + offset
    if state["residual"] is not None:
        z = z + state["residual"].float().view(shape)
    got = {"y": _activate(z, case["activation"]).to(out).view(state["x"].shape)}
    if case["train"]:
        dz = state["grad"].float().view(shape) * _slope(z, case["activation"])
        by_scale, by_offset = (dz * x).sum(1), dz.sum(1)
        got["dscale"] = by_scale.sum(0).view(-1).to(state["scale"].dtype)
        got["doffset"] = by_offset.sum(0).view(-1).to(state["offset"].dtype)
        first = (by_offset * scale).sum(2).view(shape[0], 1, shape[2], 1) / count
        second = (by_scale * scale).sum(2).view(shape[0], 1, shape[2], 1) / count
        got["dx"] = (root * (dz * scale - first - x * second)).to(out).view(state["x"].shape)
        if state["residual"] is not None:
            got["dresidual"] = dz.to(out).view(state["x"].shape)
    return got


def _keep(count, rate, seed, offset):
    """Which of `count` values are kept: 16 bits each of Philox 4x32 with 10 rounds (Salmon et al., "Parallel random numbers: as easy as
    1, 2, 3"), eight values to a counter, against the rate in units of 2^-16."""
    low = 0xFFFFFFFF
    at = torch.arange((count + 7) // 8, device=DEVICE)
    c = [at & low, at >> 32, torch.full_like(at, offset & low), torch.full_like(at, offset >> 32 & low)]
    k = [seed & low, seed >> 32 & low]
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32 & low) ^ c[1] ^ k[0], q & low, (p >> 32 & low) ^ c[3] ^ k[1], p & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    words = torch.stack(c, 1).view(-1, 4, 1)
    bits = torch.cat((words & 0xFFFF, words >> 16), 2).view(-1)
    return bits[:count] >= _share(rate)


def _share(rate):
    return math.floor(rate * 65536 + 0.5)


def _plain_dropout(state):
    case, x = state["case"], state["x"]
    keep = _keep(x.numel(), case["rate"], state["seed"], state["offset"]).view(x.shape)
    factor = 65536.0 / (65536 - _share(case["rate"]))
    zero = torch.zeros((), device=DEVICE)
    y = torch.where(keep, x.float() * factor, zero)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return {"y": y.to(x.dtype), "dx": torch.where(keep, state["grad"].float() * factor, zero).to(x.dtype)}


def _plain_dense_8bit(state):
    case, x = state["case"], state["x"]
    codes, scales = _quantize(x, 1)
    a = codes.float() * scales.repeat_interleave(BLOCK, 1)[:, :case["inputs"]]
    kernel = state["codes"].float() * state["scales"].repeat_interleave(BLOCK, 0)[:case["units"]].repeat_interleave(BLOCK, 1)[:, :case["inputs"]]
    z = a @ kernel.t()
    if state["bias"] is not None:
        z += state["bias"].float()
    if state["residual"] is not None:
        z += state["residual"].float()
    return {"y": _activate(z, case["activation"]).to(x.dtype)}


# ---------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------
def _own(state):
    import tf_approximate_b200 as ax
    case = state["case"]
    activation = None if case.get("activation", "none") == "none" else case["activation"]
    if case["op"] == "group_norm":
        x, groups, scale, offset, residual = state["x"], case["groups"], state["scale"], state["offset"], state["residual"]
        if not case["train"]:
            return {"y": ax.group_norm(x, groups, scale, offset, residual, activation, EPSILON)}
        y, statistics = ax.group_norm_forward(x, groups, scale, offset, residual, activation, EPSILON)
        dx, dscale, doffset, dresidual = ax.group_norm_backward(state["grad"], x, statistics, groups, scale, offset, residual, activation)
        got = {"y": y, "dx": dx, "dscale": dscale, "doffset": doffset}
        if residual is not None:
            got["dresidual"] = dresidual
        return got
    if case["op"] == "dropout":
        where = (case["rate"], state["seed"], state["offset"])
        return {"y": ax.dropout(state["x"], *where, residual=state["residual"]), "dx": ax.dropout(state["grad"], *where)}
    return {"y": ax.dense_8bit(state["x"], state["codes"], state["scales"], state["bias"], state["residual"], activation)}


def run(state):
    if own:
        return _own(state)
    return {"group_norm": _plain_group_norm, "dropout": _plain_dropout, "dense_8bit": _plain_dense_8bit}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------
def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "group_norm":
        n, channels = case["samples"] * case["height"] * case["width"] * case["channels"], case["channels"]
        tensors = 2 + case["residual"] + (2 + case["residual"]) * case["train"]
        params = channels * TYPES[case["params"]].itemsize * (4 if case["train"] else 2)
        return {"bytes": n * size * tensors + params, "flops": n * (24 if case["train"] else 8)}
    if case["op"] == "dropout":
        n = case["rows"] * case["columns"]
        return {"bytes": n * size * (4 + case["residual"]), "flops": 2 * n}
    t, k, n = case["rows"], case["inputs"], case["units"]
    extra = (n if case["bias"] else 0) + (t * n if case["residual"] else 0)
    return {"bytes": size * (t * k + t * n + extra) + n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK), "flops": 2 * t * k * n}


# ---------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------
_ACTIVATIONS = {"none": lambda v: v * 1.0, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}


def _exact_group_norm(case, s):
    x = s["x"].double().requires_grad_(case["train"])
    scale, offset = (s[k].double().requires_grad_(case["train"]) for k in ("scale", "offset"))
    parts = x.view(case["samples"], case["height"] * case["width"], case["groups"], -1)
    var, mean = torch.var_mean(parts, (1, 3), correction=0, keepdim=True)
    z = ((parts - mean) / torch.sqrt(var + EPSILON)).reshape(x.shape) * scale + offset
    if s["residual"] is not None:
        z = z + s["residual"].double()
    y = _ACTIVATIONS[case["activation"]](z)
    got = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, (x, scale, offset, z), s["grad"].double())
        got.update(zip(("dx", "dscale", "doffset"), grads))
        if s["residual"] is not None:
            got["dresidual"] = grads[3]
    return got


def _words(count, seed, offset):
    """The generator's words once more, in numpy's unsigned types."""
    index = np.arange(-(-count // 8), dtype=np.uint64)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    a, b, c, d = index & low, index >> half, np.uint64(offset & 0xFFFFFFFF), np.uint64(offset >> 32)
    u, v = seed & 0xFFFFFFFF, seed >> 32
    for r in range(10):
        e, f = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (f >> half) ^ b ^ np.uint64((u + r * 0x9E3779B9) % 2 ** 32), f & low, (e >> half) ^ d ^ np.uint64((v + r * 0xBB67AE85) % 2 ** 32), e & low
    return np.stack([w.astype(np.uint32) for w in (a, b, c, d)], 1).view(np.uint16).reshape(-1)[:count]


def _exact_dropout(case, s):
    share = math.floor(case["rate"] * 65536 + 0.5)
    dropped = torch.from_numpy(_words(s["x"].numel(), s["seed"], s["offset"]) < share).to(DEVICE).view(s["x"].shape)
    y, dx = (s[k].double().masked_fill_(dropped, 0.0) * (65536 / (65536 - share)) for k in ("x", "grad"))
    return {"y": y if s["residual"] is None else y + s["residual"].double(), "dx": dx}


def _exact_dense_8bit(case, s):
    x = _blocks(s["x"].double(), 1)
    top = x.abs().amax(3, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -140) / 448)).clamp(min=-126))
    scale = torch.where(top > 448 * scale, 2 * scale, torch.where(top <= 224 * scale, scale / 2, scale)).clamp(min=2.0 ** -126)
    parts = x / scale
    # e4m3: three bits behind the leading one, steps of 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(parts.abs().clamp(min=2.0 ** -6))) - 3)
    x = (torch.round(parts / step) * step * scale).view(case["rows"], -1)[:, :case["inputs"]]
    part = s["scales"].double()[:, None, :, None]
    kernel = (_blocks(s["codes"].double(), BLOCK) * part).view(part.shape[0] * BLOCK, -1)[:case["units"], :case["inputs"]]
    z = torch.einsum("tk,uk->tu", x, kernel)
    for more in (s["bias"], s["residual"]):
        if more is not None:
            z = z + more.double()
    return {"y": _ACTIVATIONS[case["activation"]](z)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"group_norm": _exact_group_norm, "dropout": _exact_dropout, "dense_8bit": _exact_dense_8bit}[case["op"]](case, s)
