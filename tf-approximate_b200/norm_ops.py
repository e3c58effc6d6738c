"""Group norm with the shortcut and the activation that follow it, and dropout without a stored mask, with their gradients: what stands between
the table convolutions and the dense layers of a network that is trained.  The reference leaves both to its host framework (Keras
GroupNormalization, Activation and Dropout); here they are kernels behind include/axconv.h.  Channels are last, as everywhere in this package."""
import torch

from . import _lib
from .dense_ops import _activation, _differentiated


def group_norm_forward(x, groups, scale=None, offset=None, residual=None, activation=None, epsilon=1e-3):
    """(y, statistics): y = activation(normalised x * scale + offset + residual), and what `group_norm_backward` needs of it.

    x [samples, ..., channels] in float32, bfloat16 or float16, any strides (other than contiguous ones are copied); its channels are a
    multiple of `groups`, and a group's mean and variance are those of its channels at all places of a sample.  scale and offset
    [channels] may be of another of these types, and are ones and zeros where None; residual has x's shape and type.  activation: None,
    "relu", "gelu" (with erf) or "silu".  Sums are fp32 and y is rounded once.  statistics [samples, groups, 2]: mean and
    1 / sqrt(variance + epsilon), in fp32."""
    return _lib.binding().group_norm_forward(x, groups, scale, offset, residual, _activation(activation), epsilon)


def group_norm_backward(grad, x, statistics, groups, scale=None, offset=None, residual=None, activation=None, need_x=True):
    """(dx, dscale, doffset, dresidual) of `group_norm_forward` for the gradient of its output; `statistics` is what it returned, the rest what it
    was given.  dscale, doffset and dresidual are there for what is given, dx where needed.  Without an activation dresidual is `grad` itself: one
    tensor, not a copy."""
    return _lib.binding().group_norm_backward(grad, x, statistics, groups, scale, offset, residual, _activation(activation), bool(need_x), True, True, True)


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, offset, residual, groups, activation, epsilon):
        y, statistics = group_norm_forward(x, groups, scale, offset, residual, activation, epsilon)
        ctx.groups, ctx.activation = groups, activation
        ctx.save_for_backward(x, scale, offset, residual, statistics)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, scale, offset, residual, statistics = ctx.saved_tensors
        return _lib.binding().group_norm_backward(grad, x, statistics, ctx.groups, scale, offset, residual, _activation(ctx.activation),
                                                  *ctx.needs_input_grad[:4]) + (None, None, None)


def group_norm(x, groups, scale=None, offset=None, residual=None, activation=None, epsilon=1e-3):
    """activation(normalised x * scale + offset + residual), differentiable once, in reverse mode; see `group_norm_forward`."""
    if _differentiated(x, scale, offset, residual):
        return _GroupNormFn.apply(x, scale, offset, residual, groups, activation, epsilon)
    return group_norm_forward(x, groups, scale, offset, residual, activation, epsilon)[0]


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rate, seed, offset):
        ctx.rate, ctx.seed = rate, seed
        ctx.offset = None if isinstance(offset, torch.Tensor) else offset
        ctx.save_for_backward(offset if ctx.offset is None else None)      # a counter that moved on before the backward pass is refused there
        return _lib.binding().dropout(x, rate, seed, offset, residual)

    @staticmethod
    def backward(ctx, grad):
        offset = ctx.saved_tensors[0] if ctx.offset is None else ctx.offset
        dx = dropout(grad, ctx.rate, ctx.seed, offset) if ctx.needs_input_grad[0] else None
        return dx, grad if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, rate, seed, offset=0, residual=None):
    """x with a share `rate` of its values set to 0 and the others divided by 1 - rate, plus residual; differentiable in reverse mode, any number of
    times.

    Which values are dropped is a function of `seed` and `offset` (ints in [0, 2^64)) and of a value's place in x alone, and is computed again for the
    gradient: no mask is stored.  Every call of a training step needs an offset (or a seed) of its own.  rate is held as a multiple of 2^-16, and the
    factor is that of the rate as it is held.  offset may be one int64 on x's device: a captured call then reads it at every replay.
    x: float32, bfloat16 or float16, any strides; residual has x's shape and type.  The gradient of x is `dropout` of y's gradient."""
    if _differentiated(x, residual):
        return _DropoutFn.apply(x, residual, rate, seed, offset)
    return _lib.binding().dropout(x, rate, seed, offset, residual)
