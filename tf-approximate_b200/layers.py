"""The layer-level caller of the op, mirroring the reference's Keras wrapper
(tf2/python/keras/layers/fake_approx_convolutional.py): per-batch min/max, fake quantisation of
input and kernel, the table convolution, then bias and activation; the backward pass is the exact
convolution's (the reference registers `conv2d_backprop_input/filter` as the gradient, :264-302)."""
import copy

import torch

from . import dense_ops, norm_ops, ops
from .ops import approx_conv2d_with_min_max_vars


def _nudge(min_v, max_v, num_bits=8):
    """TensorFlow fake-quant range nudging (restated in the reference at tf2/src/approx_ops_types.h:29-49), in fp32
    like the op.  Works on 0-d tensors of any device, so nothing is synchronised with the host.  Returns tensors
    (nudged_min, nudged_max, scale); a zero range gives zeros (tf2/src/approx_ops_types.h:135-152)."""
    f32 = torch.float32
    mn = torch.as_tensor(min_v, dtype=f32)
    mx = torch.as_tensor(max_v, dtype=f32).to(mn.device)
    qmin = torch.zeros((), dtype=f32, device=mn.device)
    qmax = torch.full((), float((1 << num_bits) - 1), dtype=f32, device=mn.device)
    zero_range = (mn == 0) & (mx == 0)
    scale = (mx - mn) / (qmax - qmin)
    safe = torch.where(zero_range, torch.ones_like(scale), scale)
    zp_from_min = qmin - mn / safe
    rounded = torch.sign(zp_from_min) * torch.floor(torch.abs(zp_from_min) + 0.5)   # half away from zero
    zp = torch.where(zp_from_min < qmin, qmin, torch.where(zp_from_min > qmax, qmax, rounded))
    nudged_min = (qmin - zp) * safe
    nudged_max = (qmax - zp) * safe
    z = torch.zeros_like(scale)
    return (torch.where(zero_range, z, nudged_min), torch.where(zero_range, z, nudged_max),
            torch.where(zero_range, z, scale))


def fake_quant_with_min_max_vars(x, min_v, max_v, num_bits=8):
    """Forward of TensorFlow's FakeQuantWithMinMaxVars: clamp to the nudged range and snap to its grid.
    The reference applies it to input and kernel before the op
    (tf2/python/keras/layers/fake_approx_convolutional.py:233-242).  min_v / max_v may be Python floats or 0-d
    tensors on x's device (then no host synchronisation happens)."""
    mn = torch.as_tensor(min_v, dtype=torch.float32).to(x.device)
    mx = torch.as_tensor(max_v, dtype=torch.float32).to(x.device)
    nmin, nmax, scale = _nudge(mn, mx, num_bits)
    zero_range = scale == 0
    inv = torch.ones((), dtype=torch.float32, device=x.device) / torch.where(zero_range, torch.ones_like(scale), scale)
    clamped = torch.minimum(torch.maximum(x, nmin), nmax)
    q = torch.floor((clamped - nmin) * inv + 0.5)
    return torch.where(zero_range, torch.zeros_like(x), q * scale + nmin)


class _FakeQuantFn(torch.autograd.Function):
    """Fake quantisation with a device-resident range (one kernel); straight-through gradient - every element lies
    inside its own tensor's range, where TensorFlow's fake-quant gradient is the identity."""

    @staticmethod
    def forward(ctx, x, range2):
        return ops.fake_quant_device_range(x, range2)

    @staticmethod
    def backward(ctx, grad):
        return grad, None


class _ColumnSumsFn(torch.autograd.Function):
    """Sums over all but the last dimension, as autograd sees them: linear, so that the gradient of a bias has derivatives."""

    @staticmethod
    def forward(ctx, x):
        ctx.shape = x.shape
        return ops.column_sums(x)

    @staticmethod
    def backward(ctx, grad):
        return grad.expand(ctx.shape)

    @staticmethod
    def jvp(ctx, tangent):
        return ops.column_sums(tangent)


def _bias_gradient(grad):
    if not torch._C._has_storage(grad):                    # batched gradients: no memory that a kernel could be given
        return grad.sum(tuple(range(grad.dim() - 1)))
    if torch.is_grad_enabled() or torch.autograd.forward_ad._current_level >= 0:
        return _ColumnSumsFn.apply(grad)
    return ops.column_sums(grad)                           # an ordinary backward pass: nobody differentiates it


class _ApproxConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, ranges, strides, padding, mul_map_file, num_bits, dilations, plan, workspace):
        ctx.save_for_backward(x, w)
        ctx.cfg = (strides, padding, dilations)
        y = approx_conv2d_with_min_max_vars(x, w, None, None, None, None, strides=strides, num_bits=num_bits,
                                            mul_map_file=mul_map_file, padding=padding, dilations=dilations,
                                            plan=plan, workspace=workspace, ranges=ranges, bias=bias)
        ctx.oshape = y.shape
        return y

    @staticmethod
    def jvp(ctx, x, w, bias, *_):
        # only a bias has a tangent here: operands with one are refused by their quantisation, which has no forward mode
        return bias.expand(ctx.oshape).contiguous()

    @staticmethod
    def backward(ctx, grad):
        x, w = ctx.saved_tensors
        strides, padding, dilations = ctx.cfg
        kh, kw = w.shape[0], w.shape[1]
        sh, sw, dh, dw = strides[1], strides[2], dilations[1], dilations[2]
        ph = pw = 0
        if padding == "SAME":
            oh, ow = -(-x.shape[1] // sh), -(-x.shape[2] // sw)
            ph = max((oh - 1) * sh + (kh - 1) * dh + 1 - x.shape[1], 0)
            pw = max((ow - 1) * sw + (kw - 1) * dw + 1 - x.shape[2], 0)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        gx = gw = gb = None
        # every step is one that autograd can differentiate again: a penalty on any of the gradients has its own gradients
        if need_x or need_w:
            # the exact convolution's two gradients, asked for as such: no forward convolution to differentiate, and a padded
            # copy only where the padding is not the same on both sides
            xc, even = x.permute(0, 3, 1, 2), ph % 2 == 0 and pw % 2 == 0
            if not even:
                xc = torch.nn.functional.pad(xc, (pw // 2, pw - pw // 2, ph // 2, ph - ph // 2))
            gx, gw, _ = torch.ops.aten.convolution_backward(
                grad.permute(0, 3, 1, 2), xc, w.permute(3, 2, 0, 1), None, (sh, sw), (ph // 2, pw // 2) if even else (0, 0), (dh, dw),
                False, (0, 0), 1, (need_x, need_w, False))
            if need_x:
                gx = gx if even else gx[:, :, ph // 2:ph // 2 + x.shape[1], pw // 2:pw // 2 + x.shape[2]]
                gx = gx.permute(0, 2, 3, 1)
            if need_w:
                gw = gw.permute(2, 3, 1, 0)
        if need_b:
            gb = _bias_gradient(grad)
        return gx, gw, gb, None, None, None, None, None, None, None, None


class FakeApproxConv2D(torch.nn.Module):
    """Conv2D whose multiplications go through a truth table
    (reference: FakeApproxConv2D, tf2/python/keras/layers/fake_approx_convolutional.py:176-261).
    Tensors are NHWC, the kernel is [KH, KW, Cin, filters]."""

    def __init__(self, in_channels, filters, kernel_size, strides=(1, 1), padding="valid", dilation_rate=(1, 1),
                 activation=None, use_bias=True, num_bits=8, mul_map_file=""):
        super().__init__()
        ks = (kernel_size, kernel_size) if isinstance(kernel_size, int) else tuple(kernel_size)
        self.strides = (strides, strides) if isinstance(strides, int) else tuple(strides)
        self.dilation_rate = (dilation_rate, dilation_rate) if isinstance(dilation_rate, int) else tuple(dilation_rate)
        self.padding = "VALID" if padding.lower() in ("valid", "causal") else padding.upper()
        self.activation = activation
        self.num_bits = num_bits
        self.mul_map_file = mul_map_file
        fan_in, fan_out = ks[0] * ks[1] * in_channels, ks[0] * ks[1] * filters
        limit = (6.0 / (fan_in + fan_out)) ** 0.5  # glorot_uniform, the Keras default
        self.kernel = torch.nn.Parameter(torch.empty(ks[0], ks[1], in_channels, filters).uniform_(-limit, limit))
        self.bias = torch.nn.Parameter(torch.zeros(filters)) if use_bias else None
        # owned by the layer, like the op instance's state in the reference: the four range scalars and the op's
        # workspace (the lookup plan of the kernel lives there between calls)
        self._ranges = None
        self._workspace = None

    def _own_buffers(self, inputs, strides4, dilations4, table):
        dev = inputs.device
        if self._ranges is None or self._ranges.device != dev:
            self._ranges = torch.empty(4, dtype=torch.float32, device=dev)
            self._workspace = None
        if ops.fast_workspace_bytes(inputs.shape, self.kernel.shape, strides4, self.padding, dilations4, table) > 0:
            return self._ranges, None            # the op's scratch for this shape holds nothing between calls
        need = ops.workspace_bytes(inputs.shape, self.kernel.shape, strides4, self.padding, dilations4)
        if self._workspace is None or self._workspace.numel() < need:
            self._workspace = torch.zeros(need, dtype=torch.uint8, device=dev)
        return self._ranges, self._workspace

    def plan_info(self):
        """{rebuilt, fallback, status, steps per mille} of the lookup plan in the layer's workspace, as the last call that used it
        left them (blocks until the current stream is idle); None where no call has: calls on the expanded tables keep none."""
        import ctypes as C
        from . import _lib
        if self._workspace is None:
            return None
        info = (C.c_int32 * 4)()
        dev = self._workspace.device
        st = _lib.load().axc_conv2d_plan_info(self._workspace.data_ptr(), info, ops._device_index(dev),
                                              C.c_void_p(torch.cuda.current_stream(dev).cuda_stream))
        ops.raise_for_status(st, "plan info")
        return {"rebuilt": int(info[0]), "fallback": int(info[1]), "status": int(info[2]), "steps_per_mille": int(info[3])}

    def forward(self, inputs):
        if self.num_bits != 8:
            raise ops.InvalidArgumentError("only num_bits == 8 is supported")
        strides4 = (1, self.strides[0], self.strides[1], 1)
        dilations4 = (1, self.dilation_rate[0], self.dilation_rate[1], 1)
        table = ops._table_for(self.mul_map_file, self.num_bits)
        ranges, workspace = self._own_buffers(inputs, strides4, dilations4, table)
        # per-batch ranges: one reduction kernel each, written where the op reads them - no host round trip
        ops.tensor_range(inputs.detach(), ranges[0:2])
        ops.tensor_range(self.kernel.detach(), ranges[2:4])
        q_in = _FakeQuantFn.apply(inputs, ranges[0:2])
        q_k = _FakeQuantFn.apply(self.kernel, ranges[2:4])
        # while the weights are being trained they change every step: no lookup plan then (nothing to rebuild)
        plan = "none" if (self.training and self.kernel.requires_grad) else "keep"
        # the op adds an fp32 bias per filter in the same pass; any other is added as torch broadcasts it
        b = self.bias
        fused = b if b is not None and b.dtype == torch.float32 and b.device == inputs.device and b.shape == self.kernel.shape[3:] else None
        y = _ApproxConvFn.apply(q_in, q_k, fused, ranges, strides4, self.padding, table, self.num_bits, dilations4,
                                plan, workspace)
        if b is not None and fused is None:
            y = y + b
        if self.activation is not None:
            y = self.activation(y)
        return y


class Dense(torch.nn.Module):
    """The exact dense layer at the end of a network of table convolutions: activation(inputs kernel + bias), in the manner of the
    Keras layer that the reference's models end with.  The kernel is [in_features, units]; inputs are cast to its type."""

    def __init__(self, in_features, units, activation=None, use_bias=True, dtype=torch.float32):
        super().__init__()
        dense_ops._activation(activation)                       # refuses an unknown name here, not at the first call
        limit = (6.0 / (in_features + units)) ** 0.5
        self.activation = activation
        self.kernel = torch.nn.Parameter(torch.empty(in_features, units).uniform_(-limit, limit).to(dtype))
        self.bias = torch.nn.Parameter(torch.zeros(units, dtype=dtype)) if use_bias else None

    def forward(self, inputs, residual=None):
        return dense_ops.dense(inputs.to(self.kernel.dtype), self.kernel, self.bias, residual, self.activation)

    def cross_entropy(self, inputs, labels, ignore_index=-100, reduction="mean"):
        """The softmax cross entropy of this layer's outputs as logits, without computing them as a tensor."""
        if self.activation not in (None, "none", "linear"):
            raise ops.InvalidArgumentError("the logits of a cross entropy have no activation")
        return dense_ops.dense_cross_entropy(inputs.to(self.kernel.dtype), self.kernel, labels, self.bias, ignore_index, reduction)


class _AnswerFn(torch.autograd.Function):
    """A result without gradients of something that has them."""

    @staticmethod
    def forward(ctx, layer, inputs, residual):
        return layer._answer(inputs, residual)

    @staticmethod
    def backward(ctx, grad):
        raise ops.InvalidArgumentError("Dense8bit has no gradients: train the Dense layer that it was made of")


class Dense8bit(torch.nn.Module):
    """A trained `Dense` layer, ready to answer in 8-bit floating point: its kernel is quantised here, once, and kept as codes [units, in_features] with
    their scales; inputs are cast to the layer's type, as `Dense` does, and quantised by the call.  It has buffers and no parameters, and no gradients: a
    backward pass through it is refused.  Casts of a network change the type of its inputs and of its bias, not what it holds in 8 bits."""

    def __init__(self, dense):
        super().__init__()
        if not isinstance(dense, Dense):
            raise ops.InvalidArgumentError("a Dense layer expected")
        self.activation, self.units, self.in_features = dense.activation, dense.kernel.shape[1], dense.kernel.shape[0]
        with torch.no_grad():
            codes, scales = dense_ops.quantize_blocks(dense.kernel.detach().t().contiguous(), rows=128)
            # rows of a multiple of 16 bytes, which the matrix kernels read where they are
            lines = torch.zeros(self.units, -(-self.in_features // 16) * 16, dtype=torch.uint8, device=codes.device)
            lines[:, :self.in_features] = codes.view(torch.uint8)
        self.register_buffer("lines", lines)
        self.register_buffer("scales", scales)
        self.register_buffer("bias", None if dense.bias is None else dense.bias.detach().clone())
        self.register_buffer("_like", torch.empty(0, dtype=dense.kernel.dtype, device=codes.device), persistent=False)       # the inputs' type

    def _apply(self, fn, recurse=True):
        # A cast of the network is not one of the codes and scales: fn has them as whole numbers, and what it makes of those but a cast is taken.
        kept = {name: self._buffers[name] for name in ("lines", "scales")}
        moved = dict(kept)
        self._buffers.update(dict.fromkeys(kept))
        try:
            super()._apply(fn, recurse)
            for name, t in kept.items():
                bits = t if name == "lines" else t.view(torch.int32)
                to = fn(bits)
                moved[name] = (to if to.dtype == bits.dtype else bits.to(to.device)).view(t.dtype)
        finally:
            self._buffers.update(moved)
        return self

    @property
    def kernel(self):
        """The codes, [units, in_features]."""
        return self.lines.view(torch.float8_e4m3fn)[:, :self.in_features]

    def _answer(self, inputs, residual):
        return dense_ops.dense_8bit(inputs.to(self._like.dtype), self.kernel, self.scales, self.bias, residual, self.activation)

    def forward(self, inputs, residual=None):
        if dense_ops._differentiated(inputs, residual):
            return _AnswerFn.apply(self, inputs, residual)
        return self._answer(inputs, residual)


class GroupNorm(torch.nn.Module):
    """Group norm of tensors with their channels last, in the manner of Keras' GroupNormalization, with the activation that follows it (and, where
    the call has one, the shortcut that is added before it): activation(normalised inputs * scale + offset + residual)."""

    def __init__(self, channels, groups=32, activation=None, epsilon=1e-3, use_scale=True, use_offset=True, dtype=torch.float32):
        super().__init__()
        dense_ops._activation(activation)                       # refuses an unknown name here, not at the first call
        if groups < 1 or channels < 1 or channels % groups:
            raise ops.InvalidArgumentError("the channels (%d) must be a multiple of the groups (%d)" % (channels, groups))
        self.groups, self.activation, self.epsilon = groups, activation, epsilon
        self.scale = torch.nn.Parameter(torch.ones(channels, dtype=dtype)) if use_scale else None
        self.offset = torch.nn.Parameter(torch.zeros(channels, dtype=dtype)) if use_offset else None

    def forward(self, inputs, residual=None):
        return norm_ops.group_norm(inputs, self.groups, self.scale, self.offset, residual, self.activation, self.epsilon)


class Dropout(torch.nn.Module):
    """Dropout without a stored mask, in the manner of the Keras layer; in evaluation the inputs pass.  `calls`, which picks the mask and counts up with
    every call in training, is an int, or with `capturable` one int64 on the inputs' device that the call itself counts up, so that a captured step
    has another mask at every replay.  seed: None for one of torch's.

    A call that a backward pass makes is one made again (torch.utils.checkpoint) and has the mask of the first time, which it is known by: every call in
    training draws a number from torch's generator of the CPU, whose state such a recomputation sets back.  Where it does not (preserve_rng_state=False),
    or the last `REMEMBERED` calls of the layer do not have it, the call is refused.

    The seed and `calls` are in the layer's state, so that a run that is taken up again has the masks that it would have had.
    copy.deepcopy makes a layer with a seed of its own where none was given: blocks that are copied drop other places."""

    REMEMBERED = 4096

    def __init__(self, rate, seed=None, capturable=False):
        super().__init__()
        if not 0.0 <= rate <= 1.0:
            raise ops.InvalidArgumentError("a rate must lie in [0, 1]")
        if seed is not None and not (isinstance(seed, int) and 0 <= seed < 1 << 64):
            raise ops.InvalidArgumentError("a seed must be an int in [0, 2^64)")
        self.rate = float(rate)
        self._draws_seed = seed is None
        self.seed = self._new_seed() if seed is None else seed
        self.capturable = capturable
        self._recent = {}                                       # number drawn from torch's generator -> offset of that call
        if capturable:
            self.register_buffer("calls", torch.zeros((), dtype=torch.int64))
        else:
            self.calls = 0

    @staticmethod
    def _new_seed():
        return torch.randint(1 << 62, (), device="cpu").item()

    def __deepcopy__(self, memo):
        other = type(self).__new__(type(self))
        memo[id(self)] = other
        other.__setstate__(copy.deepcopy(self.__getstate__(), memo))
        if self._draws_seed:
            other.seed = self._new_seed()
        return other

    def __getstate__(self):
        return dict(super().__getstate__(), _recent={})

    def __setstate__(self, state):
        super().__setstate__({"_draws_seed": False, **state, "_recent": {}})

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "seed"] = torch.tensor(self.seed - (self.seed >> 63 << 64), dtype=torch.int64)        # its 64 bits
        if not self.capturable:
            destination[prefix + "calls"] = torch.tensor(self.calls, dtype=torch.int64)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        own, rest = {}, dict(state_dict)
        for name in ("seed",) if self.capturable else ("seed", "calls"):
            t = rest.pop(prefix + name, None)                   # (states from before there were any have none)
            if t is None:
                continue
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int64 or t.dim() != 0:
                error_msgs.append("%s%s must be one int64" % (prefix, name))
                return
            own[name] = int(t) % (1 << 64)
        super()._load_from_state_dict(rest, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        self.__dict__.update(own)

    def _offset(self):
        drawn = torch.randint(1 << 62, (), device="cpu").item()
        if torch._C._current_graph_task_id() != -1:             # inside a backward pass
            if drawn not in self._recent:
                raise ops.InvalidArgumentError("dropout is run again in a backward pass that has not set torch's random state back to that of the first time")
            return self._recent[drawn]
        if self.capturable:
            offset = self.calls.clone()                         # the backward pass reads this call's own
            self.calls.add_(1)
        else:
            offset = self.calls
            self.calls += 1
        self._recent.pop(drawn, None)
        self._recent[drawn] = offset
        if len(self._recent) > self.REMEMBERED:
            del self._recent[next(iter(self._recent))]
        return offset

    def forward(self, inputs, residual=None):
        if not self.training:
            if residual is None:
                return inputs
            if not isinstance(residual, torch.Tensor) or (residual.dtype, residual.device, residual.shape) != (inputs.dtype, inputs.device, inputs.shape):
                raise ops.InvalidArgumentError("residual must be a tensor of the inputs' type, shape and device")
            return inputs + residual
        return norm_ops.dropout(inputs, self.rate, self.seed, self._offset(), residual)
