"""The exact dense layer and the cross entropy of a dense classifier, with their gradients: the exact end of a network whose
convolutions go through a truth table.  The reference takes both from its host framework (Keras Dense, sparse softmax cross
entropy with logits); here they are matrix kernels on the tensor cores behind include/axconv.h."""
import torch
from torch.autograd import forward_ad

from . import _lib
from .errors import InvalidArgumentError

_ACTIVATIONS = {None: 0, "none": 0, "linear": 0, "relu": 1, "gelu": 2, "silu": 3}
_REDUCTIONS = {"mean": 0, "sum": 1}


def _differentiated(*tensors):
    """Whether autograd has to see the call: a gradient may be asked for, or tensors may have tangents of forward mode, which the autograd
    functions refuse (they have no rule for it) and a direct call would drop."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if getattr(t, "requires_grad", False):
                return True
    return False


def _activation(name):
    if name not in _ACTIVATIONS:
        raise InvalidArgumentError("activation must be None, 'relu', 'gelu' or 'silu'")
    return _ACTIVATIONS[name]


def dense_forward(x, kernel, bias=None, residual=None, activation=None, check=False):
    """(y, kept): y = activation(x kernel + bias + residual), and what `dense_backward` needs of it.

    x [..., inputs] and kernel [inputs, units] have one type (float32, bfloat16 or float16) and any strides: a kernel that lies as
    [units, inputs] is handed over as its transpose, without a copy.  bias [units] may be of another of these types; residual has y's
    shape and type.  activation: None, "relu", "gelu" (with erf) or "silu".  Sums are fp32 and y is rounded once; fp32 operands keep
    fp32's precision.  `kept` is y for relu, the activation's argument for gelu and silu (in y's type), else None.
    check: wait for the call and raise InternalError if a wait inside the kernels ran out."""
    return _lib.binding().dense_forward(x, kernel, bias, residual, _activation(activation), bool(check))


def dense_backward(grad, x, kernel, kept=None, activation=None, bias=None, residual=None, need_x=True, need_kernel=True, check=False):
    """(dx, dkernel, dbias, dresidual) of `dense_forward` for the gradient of its output; `kept` is what it returned.  dbias and
    dresidual are there for the bias and the residual that are given (of which only type and shape count), dx and dkernel where
    needed.  dkernel lies in memory as the kernel does."""
    return _lib.binding().dense_backward(grad, x, kernel, kept, _activation(activation), bias, residual, bool(need_x), bool(need_kernel), bool(check))


class _DenseFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, bias, residual, activation):
        y, kept = dense_forward(x, kernel, bias, residual, activation)
        ctx.activation = activation
        ctx.save_for_backward(x, kernel, bias, residual, kept)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, kernel, bias, residual, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dkernel, dbias, dresidual = dense_backward(grad, x, kernel, kept, ctx.activation, bias if need[2] else None, residual if need[3] else None,
                                                       need[0], need[1])
        return dx, dkernel, dbias, dresidual, None


def dense(x, kernel, bias=None, residual=None, activation=None):
    """activation(x kernel + bias + residual), differentiable once, in reverse mode; see `dense_forward`.  Does not wait for the call: only
    `dense_forward` and `dense_backward` with `check` ask whether a wait inside the kernels ran out."""
    if _differentiated(x, kernel, bias, residual):
        return _DenseFn.apply(x, kernel, bias, residual, activation)
    return _lib.binding().dense_forward(x, kernel, bias, residual, _activation(activation), None)[0]


def _entropy(x, kernel, labels, bias, ignore_index, reduction, grad_scale, scratch_limit, row_losses, need, check):
    if reduction not in _REDUCTIONS:
        raise InvalidArgumentError("reduction must be 'mean' or 'sum'")
    return _lib.binding().entropy(x, kernel, labels, bias, int(ignore_index), _REDUCTIONS[reduction], float(grad_scale), int(scratch_limit or 0), row_losses,
                                  *map(bool, need), check)


def dense_cross_entropy_gradients(x, kernel, labels, bias=None, ignore_index=-100, reduction="mean", grad_scale=1.0, scratch_limit=None, check=False):
    """(loss, dx, dkernel, dbias) of the softmax cross entropy of a dense classifier, in one call and without keeping its logits.

    x [..., inputs] and kernel [inputs, classes] as for `dense_forward`, labels int64 [...].  Rows with the label `ignore_index` take
    no part; the loss is the mean or the sum over the others (0 if there is none), a fp32 scalar.  The gradients are those of
    grad_scale * loss, in the operands' types (dbias in the bias's); dbias is None without a bias.  A label that is neither a class nor
    ignore_index makes the loss and the gradients NaN.
    scratch_limit: bytes of scratch in which the exponentials may be kept (default 4 GiB); where they do not fit, the logits are
    computed a second time, in pieces of the classes."""
    loss, _, dx, dkernel, dbias = _entropy(x, kernel, labels, bias, ignore_index, reduction, grad_scale, scratch_limit, False, (True, True, True), bool(check))
    return loss, dx, dkernel, dbias


class _EntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, bias, labels, ignore_index, reduction, scratch_limit):
        loss, _, dx, dkernel, dbias = _entropy(x, kernel, labels, bias, ignore_index, reduction, 1.0, scratch_limit, False, ctx.needs_input_grad[:3], False)
        ctx.save_for_backward(dx, dkernel, dbias)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        # fp32 products, rounded once (torch would round the factor to the gradients' type first)
        return _lib.binding().scaled(grad, *ctx.saved_tensors) + (None,) * 4


def dense_cross_entropy(x, kernel, labels, bias=None, ignore_index=-100, reduction="mean", row_losses=False, scratch_limit=None):
    """Softmax cross entropy of a dense classifier; see `dense_cross_entropy_gradients`.  Differentiable once, in reverse mode: the gradients
    are computed with the loss and kept, in the operands' types, until backward multiplies them by its fp32 factor, so that small gradients of
    float16 operands are lost before a loss scale reaches them (`dense_cross_entropy_gradients` has one that comes before that rounding).  row_losses: (loss, the rows' own losses), without gradients."""
    if not row_losses and _differentiated(x, kernel, bias):
        return _EntropyFn.apply(x, kernel, bias, labels, ignore_index, reduction, scratch_limit)
    loss, rows, _, _, _ = _entropy(x, kernel, labels, bias, ignore_index, reduction, 1.0, scratch_limit, bool(row_losses), (False, False, False), False)
    return (loss, rows) if row_losses else loss
