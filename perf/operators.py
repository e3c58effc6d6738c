"""The operators that train and serve the exact end of a network of table convolutions, with the sizes that performance is
measured at: the dense layer (matrix product with bias, residual and activation) with its gradients, the cross entropy of a
dense classifier with its gradients, and the AdamW step over all tensors of a network.

A case is one pass through an operator.  With `own` false, `run` computes it in elementary torch operations in fp32, rounded
once at the end to the type of its output; with `own` true, by the calls of this package.  Sizes are those of the heads and
parameter lists of the ResNet-50 and ResNet-20 workloads, and generic ones; `draw` gives more cases of the same ranges."""
import math

import torch

own = False

DEVICE = torch.device("cuda", 0)
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 256            # values of an optimizer state that share a scale; every tensor's state starts at a multiple of it
IGNORE = -100


# ---------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------
def dense(rows, inputs, units, dtype, activation="none", bias=True, residual=False, train=False, order="in_out"):
    return {"op": "dense", "rows": rows, "inputs": inputs, "units": units, "dtype": dtype, "activation": activation, "bias": bias,
            "residual": residual, "train": train, "order": order}


def entropy(rows, inputs, classes, dtype, bias=False, ignored=0.0, order="in_out"):
    return {"op": "entropy", "rows": rows, "inputs": inputs, "classes": classes, "dtype": dtype, "bias": bias, "ignored": ignored,
            "order": order}


def adamw(net, dtype, bits, size=0, tensors=0):
    return {"op": "adamw", "net": net, "dtype": dtype, "bits": bits, "size": size, "tensors": tensors}


def listed():
    return [
        # one row through a wide layer, as a model answers token by token: the weights are read once, latency counts
        dict(dense(1, 4096, 16384, "bfloat16", "silu", bias=False, order="out_in"), name="dense_one_row"),
        # the classifier of ResNet-50 at the benchmark's batch, in the type that the table convolutions work in: a training step
        dict(dense(256, 2048, 1000, "float32", train=True), name="dense_resnet50_head"),
        # sizes that are multiples of nothing, a shortcut and a ReLU: a training step
        dict(dense(1531, 1030, 2777, "float16", "relu", residual=True, train=True, order="out_in"), name="dense_ragged"),
        # the widening layer of a large block at a training batch: bound by the matrix units
        dict(dense(8192, 4096, 16384, "bfloat16", "gelu", train=True), name="dense_large"),
        # the classifier of ResNet-20 at its batch: ten classes, a pass is mostly latency
        dict(entropy(1024, 64, 10, "float32", bias=True), name="entropy_resnet20_head"),
        # the classifier of ResNet-50 at its batch
        dict(entropy(256, 2048, 1000, "bfloat16", bias=True), name="entropy_resnet50_head"),
        # a vocabulary of odd size, a fifth of the rows without a label
        dict(entropy(2047, 1024, 50001, "bfloat16", bias=True, ignored=0.2, order="out_in"), name="entropy_ragged"),
        # a large vocabulary at a training batch
        dict(entropy(8192, 2048, 131072, "bfloat16", order="out_in"), name="entropy_large"),
        # every parameter of ResNet-20 (65 small tensors): a pass is mostly latency
        dict(adamw("resnet20", "float32", 32), name="adamw_resnet20"),
        # every parameter of ResNet-50 (161 tensors, 25.6 million values)
        dict(adamw("resnet50", "float32", 32), name="adamw_resnet50"),
        # the same with states in 8 bits
        dict(adamw("resnet50", "float32", 8), name="adamw_resnet50_8bit"),
        # half a billion values in two bytes with states in 8 bits, in tensors of unequal and odd sizes
        dict(adamw("mixed", "bfloat16", 8, size=1 << 29, tensors=48), name="adamw_large_8bit"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("dense", "entropy", "adamw"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    order = rng.choice(("in_out", "out_in"))
    if op == "dense":
        train = rng.random() < 0.6
        rows, inputs, units = _log(rng, 16 if train else 1, 8192), _log(rng, 48, 4096), _log(rng, 40, 16384)
        return dense(rows, inputs, units, dtype, rng.choice(("none", "relu", "gelu", "silu")), rng.random() < 0.7, rng.random() < 0.4, train, order)
    if op == "entropy":
        rows, inputs = _log(rng, 64, 8192), _log(rng, 64, 2048)
        classes = _log(rng, 10, 131072)
        if dtype == "float32":                       # six times the products: no fp32 case above a sixteenth of the largest
            classes = max(10, min(classes, (1 << 27) // rows))
        return entropy(rows, inputs, classes, dtype, rng.random() < 0.4, rng.choice((0.0, 0.0, 0.1, 0.5)), order)
    bits = rng.choice((32, 8))
    if rng.random() < 0.3:
        return adamw(rng.choice(("resnet20", "resnet50")), dtype, bits)
    return adamw("mixed", dtype, bits, _log(rng, 1 << 14, 1 << (26 if dtype == "float32" else 28)), _log(rng, 2, 200))


# ---------------------------------------------------------------------------------------------------
# shapes of the parameter lists
# ---------------------------------------------------------------------------------------------------
def _with_norm(shape):
    return [shape, (shape[-1],), (shape[-1],)]          # a convolution, and scale and offset of its channels


def parameter_shapes(case):
    if case["net"] == "resnet20":
        got, cin = _with_norm((3, 3, 3, 16)), 16
        for width in (16, 32, 64):
            for block in range(3):
                got += _with_norm((3, 3, cin, width)) + _with_norm((3, 3, width, width))
                if cin != width:
                    got += _with_norm((1, 1, cin, width))
                cin = width
        return got + [(64, 10), (10,)]
    if case["net"] == "resnet50":
        got, cin = _with_norm((7, 7, 3, 64)), 64
        for width, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
            for block in range(blocks):
                got += _with_norm((1, 1, cin, width)) + _with_norm((3, 3, width, width)) + _with_norm((1, 1, width, 4 * width))
                if block == 0:
                    got += _with_norm((1, 1, cin, 4 * width))
                cin = 4 * width
        return got + [(2048, 1000), (1000,)]
    # unequal tensors: a few hold most of the values, many are short
    weights = [0.55 ** (i % 12) for i in range(case["tensors"])]
    total = sum(weights)
    return [(max(1, int(case["size"] * w / total) + (i * 37) % 11 - 5),) for i, w in enumerate(weights)]


def _numel(shape):
    return math.prod(shape)


def _padded(shape):
    return -(-_numel(shape) // BLOCK) * BLOCK


# ---------------------------------------------------------------------------------------------------
# what a user's program has in hand
# ---------------------------------------------------------------------------------------------------
def _normal(g, shape, scale, dtype):
    return (torch.randn(shape, device=DEVICE, generator=g) * scale).to(dtype)


def _kernel(g, inputs, units, order, dtype):
    """[inputs, units], stored in that order or, as tied embeddings are, the other way round."""
    if order == "in_out":
        return _normal(g, (inputs, units), inputs ** -0.5, dtype)
    return _normal(g, (units, inputs), inputs ** -0.5, dtype).t()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    if case["op"] == "dense":
        rows, inputs, units = case["rows"], case["inputs"], case["units"]
        return {"case": case, "x": _normal(g, (rows, inputs), 1.0, dtype), "kernel": _kernel(g, inputs, units, case["order"], dtype),
                "bias": _normal(g, (units,), 0.1, dtype) if case["bias"] else None,
                "residual": _normal(g, (rows, units), 1.0, dtype) if case["residual"] else None,
                "grad": _normal(g, (rows, units), 0.05, dtype) if case["train"] else None}
    if case["op"] == "entropy":
        rows, inputs, classes = case["rows"], case["inputs"], case["classes"]
        x = _normal(g, (rows, inputs), 2.0, dtype)
        kernel = _kernel(g, inputs, classes, case["order"], dtype)
        # half of the labels are what the model would answer among a few, as in a model that has learned something
        labels = torch.randint(classes, (rows,), device=DEVICE, generator=g)
        other = torch.randint(classes, (8,), device=DEVICE, generator=g)
        best = other[(x.float() @ kernel[:, other].float()).argmax(1)]
        labels = torch.where(torch.rand(rows, device=DEVICE, generator=g) < 0.5, best, labels)
        labels = torch.where(torch.rand(rows, device=DEVICE, generator=g) < case["ignored"], torch.full_like(labels, IGNORE), labels)
        # gradients in float16 are scaled, as in mixed-precision training: most of them would be zeros in that type
        return {"case": case, "x": x, "kernel": kernel, "labels": labels, "scale": 4096.0 if dtype == torch.float16 else 1.0,
                "bias": _normal(g, (classes,), 0.1, dtype) if case["bias"] else None}
    shapes = parameter_shapes(case)
    total = sum(_padded(s) for s in shapes)
    flat = (torch.randn(total, device=DEVICE, generator=g) * 0.05).to(dtype)
    # gradients of very different size from block to block, some of them zero (a unit that never answered)
    scale = torch.exp(torch.randn(total // BLOCK, 1, device=DEVICE, generator=g) * 2.0 - 5.0)
    grads = torch.randn(total // BLOCK, BLOCK, device=DEVICE, generator=g) * scale
    grads *= torch.rand(total // BLOCK, BLOCK, device=DEVICE, generator=g) > 0.05
    grads = grads.view(-1).to(dtype)
    state = {"case": case, "flat": flat, "flat_grads": grads, "params": [], "grads": [], "step": 0,
             "options": {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}}
    at = 0
    for s in shapes:
        n = _numel(s)
        state["params"].append(flat[at:at + n].view(s))
        state["grads"].append(grads[at:at + n].view(s))
        flat[at + n:at + _padded(s)] = 0
        grads[at + n:at + _padded(s)] = 0
        at += _padded(s)
    if own:
        import tf_approximate_b200 as ax
        state["optimizer"] = ax.AdamW(state["params"], state_bits=case["bits"], **state["options"])
    elif case["bits"] == 32:
        state["exp_avg"] = torch.zeros(total, device=DEVICE)
        state["exp_avg_sq"] = torch.zeros(total, device=DEVICE)
    else:
        state["exp_avg"] = torch.zeros(total, device=DEVICE).to(torch.float8_e4m3fn)
        state["exp_avg_sq_root"] = torch.zeros(total, device=DEVICE).to(torch.float8_e4m3fn)
        state["exp_avg_scale"] = torch.zeros(total // BLOCK, device=DEVICE)
        state["exp_avg_sq_root_scale"] = torch.zeros(total // BLOCK, device=DEVICE)
    return state


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
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * 0.7071067811865476)) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain_dense(state):
    case, x, kernel = state["case"], state["x"].float(), state["kernel"].float()
    out = state["x"].dtype
    z = x @ kernel
    if state["bias"] is not None:
        z += state["bias"].float()
    if state["residual"] is not None:
        z += state["residual"].float()
    got = {"y": _activate(z, case["activation"]).to(out)}
    if case["train"]:
        dz = state["grad"].float() * _slope(z, case["activation"])
        got["dx"] = (dz @ kernel.t()).to(out)
        got["dkernel"] = (x.t() @ dz if case["order"] == "in_out" else (dz.t() @ x).t()).to(out)
        if state["bias"] is not None:
            got["dbias"] = dz.sum(0).to(out)
        if state["residual"] is not None:
            got["dresidual"] = dz.to(out)
    return got


def _plain_entropy(state):
    case, x, kernel, labels = state["case"], state["x"].float(), state["kernel"].float(), state["labels"]
    out = state["x"].dtype
    logits = x @ kernel
    if state["bias"] is not None:
        logits += state["bias"].float()
    valid = labels != IGNORE
    count = valid.sum().clamp(min=1).float()
    rows, at = torch.arange(labels.numel(), device=labels.device), labels.clamp(min=0)
    top = logits.amax(1, keepdim=True)
    target = logits[rows, at] - top[:, 0]
    logits = torch.exp(logits.sub_(top))                 # from here on: exponentials, then the gradient of the logits
    total = logits.sum(1)
    losses = torch.where(valid, torch.log(total) - target, torch.zeros_like(total))
    share = valid.float() * (state["scale"] / count)
    logits *= (share / total)[:, None]
    logits[rows, at] -= share
    got = {"loss": losses.sum() / count, "dx": (logits @ kernel.t()).to(out),
           "dkernel": (x.t() @ logits if case["order"] == "in_out" else (logits.t() @ x).t()).to(out)}
    if state["bias"] is not None:
        got["dbias"] = logits.sum(0).to(out)
    return got


def _encode(x, smallest):
    """Codes of 8 bits with a scale for each block; `smallest`: a value above zero keeps a code above zero."""
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1) / 448.0
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    part = x / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    part = torch.where(scale[:, None] > 0, part, torch.zeros_like(part))
    if smallest:
        part = torch.where(part > 0, part.clamp(min=2.0 ** -9), part)
    return part.to(torch.float8_e4m3fn).view(-1), scale


def _plain_adamw(state):
    o, b1, b2 = state["options"], *state["options"]["betas"]
    state["step"] += 1
    p, g = state["flat"].float(), state["flat_grads"].float()
    if state["case"]["bits"] == 32:
        m, v = state["exp_avg"], state["exp_avg_sq"]
    else:
        m = (state["exp_avg"].float().view(-1, BLOCK) * state["exp_avg_scale"][:, None]).view(-1)
        r = (state["exp_avg_sq_root"].float().view(-1, BLOCK) * state["exp_avg_sq_root_scale"][:, None]).view(-1)
        v = r * r
    m = m + (1.0 - b1) * (g - m)
    v = v + (1.0 - b2) * (g * g - v)
    c1, c2 = 1.0 - b1 ** state["step"], 1.0 - b2 ** state["step"]
    p = p * (1.0 - o["lr"] * o["weight_decay"]) - (o["lr"] / c1) * m / (torch.sqrt(v) / math.sqrt(c2) + o["eps"])
    state["flat"].copy_(p)
    if state["case"]["bits"] == 32:
        state["exp_avg"], state["exp_avg_sq"] = m, v
        return {"params": state["flat"], "exp_avg": m, "exp_avg_sq": v}
    state["exp_avg"], state["exp_avg_scale"] = _encode(m, False)
    state["exp_avg_sq_root"], state["exp_avg_sq_root_scale"] = _encode(torch.sqrt(v), True)
    return {"params": state["flat"], **{k: state[k] for k in ("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale")}}


# ---------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------
def _own(state):
    import tf_approximate_b200 as ax
    case = state["case"]
    if case["op"] == "dense":
        activation = None if case["activation"] == "none" else case["activation"]
        if not case["train"]:
            return {"y": ax.dense(state["x"], state["kernel"], state["bias"], state["residual"], activation)}
        y, kept = ax.dense_forward(state["x"], state["kernel"], state["bias"], state["residual"], activation)
        dx, dkernel, dbias, dresidual = ax.dense_backward(state["grad"], state["x"], state["kernel"], kept, activation,
                                                          bias=state["bias"], residual=state["residual"])
        got = {"y": y, "dx": dx, "dkernel": dkernel}
        if dbias is not None:
            got["dbias"] = dbias
        if dresidual is not None:
            got["dresidual"] = dresidual
        return got
    if case["op"] == "entropy":
        loss, dx, dkernel, dbias = ax.dense_cross_entropy_gradients(state["x"], state["kernel"], state["labels"], state["bias"],
                                                                    ignore_index=IGNORE, grad_scale=state["scale"])
        got = {"loss": loss, "dx": dx, "dkernel": dkernel}
        if dbias is not None:
            got["dbias"] = dbias
        return got
    o = state["optimizer"]
    o.step(state["grads"])
    if case["bits"] == 32:
        return {"params": state["flat"], "exp_avg": o.exp_avg, "exp_avg_sq": o.exp_avg_sq}
    return {"params": state["flat"], "exp_avg": o.exp_avg, "exp_avg_scale": o.exp_avg_scale,
            "exp_avg_sq_root": o.exp_avg_sq_root, "exp_avg_sq_root_scale": o.exp_avg_sq_root_scale}


def run(state):
    if own:
        return _own(state)
    return {"dense": _plain_dense, "entropy": _plain_entropy, "adamw": _plain_adamw}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------
def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "adamw":
        n = sum(_numel(s) for s in parameter_shapes(case))
        # parameter, gradient and two states read, parameter and states written; a scale of each state for 256 values
        states = 16 if case["bits"] == 32 else 4 + 4 * 4 / BLOCK
        return {"bytes": n * (3 * size + states), "flops": 14 * n}
    t, k = case["rows"], case["inputs"]
    if case["op"] == "dense":
        n = case["units"]
        extra = (n if case["bias"] else 0) + (t * n if case["residual"] else 0)
        reads, writes, products = t * k + k * n + extra, t * n, 2
        if case["train"]:
            reads, writes, products = reads + t * n, writes + t * k + k * n + extra, 6
        return {"bytes": size * (reads + writes), "flops": products * t * k * n}
    n = case["classes"]
    return {"bytes": size * 2 * (t * k + k * n + (n if case["bias"] else 0)) + 8 * t, "flops": 6 * t * k * n}


# ---------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------
def _exact_dense(case, s):
    x, kernel = s["x"].double(), s["kernel"].double()
    z = torch.zeros(case["rows"], case["units"], dtype=torch.float64, device=DEVICE)
    for part in (s["bias"], s["residual"]):
        if part is not None:
            z = z + part.double()
    z = torch.addmm(z, x, kernel)
    z.requires_grad_(case["train"])
    act = {"none": lambda v: v * 1.0, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}
    y = act[case["activation"]](z)
    got = {"y": y.detach()}
    if case["train"]:
        dz, = torch.autograd.grad(y, z, s["grad"].double())
        got["dx"] = torch.einsum("tn,kn->tk", dz, kernel)
        got["dkernel"] = torch.einsum("tk,tn->kn", x, dz)
        if s["bias"] is not None:
            got["dbias"] = dz.sum(0)
        if s["residual"] is not None:
            got["dresidual"] = dz
    return got


def _exact_entropy(case, s):
    x, kernel, labels = s["x"].double(), s["kernel"].double(), s["labels"]
    has = torch.nonzero(labels != IGNORE)[:, 0]
    share = 1.0 / max(1, has.numel())
    got = {"loss": torch.zeros((), dtype=torch.float64, device=DEVICE), "dx": torch.zeros_like(x), "dkernel": torch.zeros_like(kernel)}
    if s["bias"] is not None:
        got["dbias"] = torch.zeros(case["classes"], dtype=torch.float64, device=DEVICE)
    for rows in has.split(2048):
        logp = x[rows] @ kernel
        if s["bias"] is not None:
            logp += s["bias"].double()
        logp -= torch.logsumexp(logp, 1, keepdim=True)
        mine = labels[rows]
        got["loss"] -= share * logp.gather(1, mine[:, None]).sum()
        d = torch.exp(logp).scatter_add_(1, mine[:, None], torch.full((rows.numel(), 1), -1.0, dtype=torch.float64, device=DEVICE))
        d *= share * s["scale"]
        got["dx"][rows] = d @ kernel.t()
        got["dkernel"] += x[rows].t() @ d
        if s["bias"] is not None:
            got["dbias"] += d.sum(0)
    return got


def _exact_adamw(case, s):
    """The first step: states are zero before it.  Codes of 8 bits have no value in 64 bits, their scales have."""
    lr, (b1, b2), eps, decay = (s["options"][k] for k in ("lr", "betas", "eps", "weight_decay"))
    p, g = s["flat"].double(), s["flat_grads"].double()
    first, second = g * (1 - b1), g * g * (1 - b2)
    p = p - lr * decay * p - lr * g / (g.abs() + eps)
    if case["bits"] == 32:
        return {"params": p, "exp_avg": first, "exp_avg_sq": second}
    return {"params": p, "exp_avg": None, "exp_avg_scale": first.abs().view(-1, BLOCK).amax(1) / 448, "exp_avg_sq_root": None,
            "exp_avg_sq_root_scale": second.sqrt().view(-1, BLOCK).amax(1) / 448}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"dense": _exact_dense, "entropy": _exact_entropy, "adamw": _exact_adamw}[case["op"]](case, s)
