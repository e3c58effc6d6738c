"""The exact dense layer and the cross entropy of a dense classifier, with their gradients: the exact end of a network whose
convolutions go through a truth table.  The reference takes both from its host framework (Keras Dense, sparse softmax cross
entropy with logits); here they are matrix kernels on the tensor cores behind include/axconv.h."""
import ctypes as C

import torch

from . import _lib
from .errors import InternalError, InvalidArgumentError, raise_for_status
from .ops import _cuda_detail

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "none": 0, "linear": 0, "relu": 1, "gelu": 2, "silu": 3}
_REDUCTIONS = {"mean": 0, "sum": 1}


def _activation(name):
    if name not in _ACTIVATIONS:
        raise InvalidArgumentError("activation must be None, 'relu', 'gelu' or 'silu'")
    return _ACTIVATIONS[name]


def _operands(x, kernel, bias):
    """x as [rows, inputs]; refuses what the kernels cannot be given."""
    if not isinstance(x, torch.Tensor) or not isinstance(kernel, torch.Tensor):
        raise InvalidArgumentError("x and kernel must be torch tensors")
    if not x.is_cuda or kernel.device != x.device:
        raise InvalidArgumentError("x and kernel must live on one CUDA device (this build has no CPU kernel)")
    if x.dtype not in _TYPES or kernel.dtype is not x.dtype:
        raise InvalidArgumentError("x and kernel must have one type, float32, bfloat16 or float16")
    if x.dim() < 1 or kernel.dim() != 2 or kernel.shape[0] != x.shape[-1]:
        raise InvalidArgumentError("x [..., inputs] and kernel [inputs, units] expected, got %s and %s" % (tuple(x.shape), tuple(kernel.shape)))
    if bias is not None and (bias.dtype not in _TYPES or bias.device != x.device or bias.shape != kernel.shape[1:]):
        raise InvalidArgumentError("bias must be a float32, bfloat16 or float16 tensor of shape (%d,) on x's device" % kernel.shape[1])
    # detach: the library is given addresses, autograd has nothing to follow here
    x2 = x.detach() if x.dim() == 2 else x.detach().reshape(-1, x.shape[-1]) if x.numel() else x.detach().reshape(x.shape[:-1].numel(), x.shape[-1])
    return x2, kernel.detach(), None if bias is None else bias.detach().contiguous()


def _other(t, name, shape, x):
    """A tensor that goes with the output, as rows of `units` values."""
    if not isinstance(t, torch.Tensor) or t.dtype is not x.dtype or t.device != x.device or t.shape != shape:
        raise InvalidArgumentError("%s must be a %s tensor of shape %s on x's device" % (name, x.dtype, tuple(shape)))
    return t.detach().reshape(shape[:-1].numel(), shape[-1])


def _pointer(t):
    return None if t is None else t.data_ptr()


def _transposed(kernel):
    """Whether the kernel lies in memory as [units, inputs]: its gradient then does too."""
    return kernel.stride(0) == 1 and kernel.stride(1) != 1


def _dense_desc(x2, kernel, bias, activation, residual_stride=0):
    return _lib.DenseDesc(x2.shape[0], x2.shape[1], kernel.shape[1], _TYPES[x2.dtype], 0 if bias is None else _TYPES[bias.dtype], _activation(activation),
                          1 if _transposed(kernel) else 0, x2.stride(0), x2.stride(1), kernel.stride(0), kernel.stride(1), residual_stride)


def _stream(x):
    return C.c_void_p(torch.cuda.current_stream(x.device).cuda_stream)


def _check_status(ws, x):
    word = C.c_int32(-1)
    raise_for_status(_lib.load().axc_matrix_status(ws.data_ptr(), C.byref(word), x.get_device(), _stream(x)), "status", _cuda_detail())
    if word.value != 0:
        raise InternalError("a wait inside a matrix kernel ran out (status %d): the result is not valid" % word.value)


def dense_forward(x, kernel, bias=None, residual=None, activation=None, check=False):
    """(y, kept): y = activation(x kernel + bias + residual), and what `dense_backward` needs of it.

    x [..., inputs] and kernel [inputs, units] have one type (float32, bfloat16 or float16) and any strides: a kernel that lies as
    [units, inputs] is handed over as its transpose, without a copy.  bias [units] may be of another of these types; residual has y's
    shape and type.  activation: None, "relu", "gelu" (with erf) or "silu".  Sums are fp32 and y is rounded once; fp32 operands keep
    fp32's precision.  `kept` is y for relu, the activation's argument for gelu and silu (in y's type), else None.
    check: wait for the call and raise InternalError if a wait inside the kernels ran out."""
    x2, k, b = _operands(x, kernel, bias)
    shape = x.shape[:-1] + k.shape[1:]
    r = None
    if residual is not None:
        r = _other(residual, "residual", shape, x)
        if r.stride(1) != 1 and r.shape[1] > 1:
            r = r.contiguous()
    desc = _dense_desc(x2, k, b, activation, 0 if r is None else r.stride(0))
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    kept = y if desc.activation == 1 else torch.empty_like(y) if desc.activation > 1 else None
    L, index = _lib.load(), x.get_device()
    size = C.c_size_t()
    raise_for_status(L.axc_dense_workspace_bytes(C.byref(desc), x2.data_ptr(), k.data_ptr(), index, C.byref(size), None), "dense", "workspace")
    ws = torch.empty(size.value, dtype=torch.uint8, device=x.device)
    st = L.axc_dense_forward(C.byref(desc), x2.data_ptr(), k.data_ptr(), _pointer(b), _pointer(r), y.data_ptr(), _pointer(kept) if desc.activation > 1 else None,
                             ws.data_ptr(), size.value, index, _stream(x))
    raise_for_status(st, "dense", _cuda_detail() if st == 100 else "")
    if check and y.numel():
        _check_status(ws, x)
    return y, kept


def dense_backward(grad, x, kernel, kept=None, activation=None, bias=None, residual=None, need_x=True, need_kernel=True, check=False):
    """(dx, dkernel, dbias, dresidual) of `dense_forward` for the gradient of its output; `kept` is what it returned.  dbias and
    dresidual are there for the bias and the residual that are given (of which only type and shape count), dx and dkernel where
    needed.  dkernel lies in memory as the kernel does."""
    x2, k, b = _operands(x, kernel, bias)
    shape = x.shape[:-1] + k.shape[1:]
    g = _other(grad, "grad", shape, x).contiguous()
    desc = _dense_desc(x2, k, b, activation)
    if desc.activation:
        kept = _other(kept, "kept", shape, x).contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
    dkernel = None
    if need_kernel:
        dkernel = torch.empty((k.shape[1], k.shape[0]) if desc.kernel_gradient_transposed else k.shape, dtype=k.dtype, device=k.device)
    dbias = torch.empty_like(b) if b is not None else None
    dresidual = None
    if residual is not None:
        _other(residual, "residual", shape, x)
        dresidual = torch.empty(shape, dtype=x.dtype, device=x.device) if desc.activation else grad
    L, index = _lib.load(), x.get_device()
    size = C.c_size_t()
    raise_for_status(L.axc_dense_workspace_bytes(C.byref(desc), x2.data_ptr(), k.data_ptr(), index, None, C.byref(size)), "dense gradients", "workspace")
    ws = torch.empty(size.value, dtype=torch.uint8, device=x.device)
    st = L.axc_dense_backward(C.byref(desc), g.data_ptr(), x2.data_ptr(), k.data_ptr(), _pointer(kept) if desc.activation else None, _pointer(dx), _pointer(dkernel),
                              _pointer(dbias), _pointer(dresidual) if desc.activation else None, ws.data_ptr(), size.value, index, _stream(x))
    raise_for_status(st, "dense gradients", _cuda_detail() if st == 100 else "")
    if check and (need_x or need_kernel):
        _check_status(ws, x)
    if dkernel is not None and desc.kernel_gradient_transposed:
        dkernel = dkernel.t()
    return dx, dkernel, dbias, dresidual


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
    """activation(x kernel + bias + residual), differentiable once; see `dense_forward`."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, kernel, bias, residual)):
        return _DenseFn.apply(x, kernel, bias, residual, activation)
    return dense_forward(x, kernel, bias, residual, activation)[0]


def _entropy(x, kernel, labels, bias, ignore_index, reduction, grad_scale, scratch_limit, row_losses, need, check):
    x2, k, b = _operands(x, kernel, bias)
    if reduction not in _REDUCTIONS:
        raise InvalidArgumentError("reduction must be 'mean' or 'sum'")
    if not isinstance(labels, torch.Tensor) or labels.dtype != torch.int64 or labels.device != x.device or labels.shape != x.shape[:-1]:
        raise InvalidArgumentError("labels must be an int64 tensor of shape %s on x's device" % (tuple(x.shape[:-1]),))
    if k.shape[0] == 0 or k.shape[1] == 0:
        raise InvalidArgumentError("a classifier needs inputs and classes")
    labels = labels.reshape(-1).contiguous()
    transposed = _transposed(k)
    desc = _lib.EntropyDesc(x2.shape[0], x2.shape[1], k.shape[1], _TYPES[x.dtype], 0 if b is None else _TYPES[b.dtype], _REDUCTIONS[reduction], 1 if transposed else 0,
                            ignore_index, scratch_limit or 0, x2.stride(0), x2.stride(1), k.stride(0), k.stride(1), grad_scale)
    dev = x.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    rows = torch.empty(labels.shape, dtype=torch.float32, device=dev) if row_losses else None
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] else None
    dkernel = torch.empty((k.shape[1], k.shape[0]) if transposed else k.shape, dtype=k.dtype, device=dev) if need[1] else None
    dbias = torch.empty_like(b) if b is not None and need[2] else None
    L, index = _lib.load(), x.get_device()
    alone, size = C.c_size_t(), C.c_size_t()
    raise_for_status(L.axc_entropy_workspace_bytes(C.byref(desc), x2.data_ptr(), k.data_ptr(), index, C.byref(alone), C.byref(size)), "dense cross entropy", "workspace")
    ws = torch.empty(size.value if dx is not None or dkernel is not None or dbias is not None else alone.value, dtype=torch.uint8, device=dev)
    st = L.axc_entropy(C.byref(desc), x2.data_ptr(), k.data_ptr(), _pointer(b), labels.data_ptr(), loss.data_ptr(), _pointer(rows), _pointer(dx), _pointer(dkernel),
                       _pointer(dbias), ws.data_ptr(), ws.numel(), index, _stream(x))
    raise_for_status(st, "dense cross entropy", _cuda_detail() if st == 100 else "")
    if check:
        _check_status(ws, x)
    if dkernel is not None and transposed:
        dkernel = dkernel.t()
    return loss, rows, dx, dkernel, dbias


def dense_cross_entropy_gradients(x, kernel, labels, bias=None, ignore_index=-100, reduction="mean", grad_scale=1.0, scratch_limit=None, check=False):
    """(loss, dx, dkernel, dbias) of the softmax cross entropy of a dense classifier, in one call and without keeping its logits.

    x [..., inputs] and kernel [inputs, classes] as for `dense_forward`, labels int64 [...].  Rows with the label `ignore_index` take
    no part; the loss is the mean or the sum over the others (0 if there is none), a fp32 scalar.  The gradients are those of
    grad_scale * loss, in the operands' types (dbias in the bias's); dbias is None without a bias.  A label that is neither a class nor
    ignore_index makes the loss and the gradients NaN.
    scratch_limit: bytes of scratch in which the exponentials may be kept (default 4 GiB); where they do not fit, the logits are
    computed a second time, in pieces of the classes."""
    loss, _, dx, dkernel, dbias = _entropy(x, kernel, labels, bias, ignore_index, reduction, grad_scale, scratch_limit, False, (True, True, True), check)
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
        return tuple(None if t is None else t * grad.to(t.dtype) for t in ctx.saved_tensors) + (None,) * 4


def dense_cross_entropy(x, kernel, labels, bias=None, ignore_index=-100, reduction="mean", row_losses=False, scratch_limit=None):
    """Softmax cross entropy of a dense classifier; see `dense_cross_entropy_gradients`.  Differentiable once: the gradients are
    computed with the loss and kept until backward, so float16 operands want a loss scale there (`dense_cross_entropy_gradients`
    has one).  row_losses: (loss, the rows' own losses), without gradients."""
    if not row_losses and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, kernel, bias)):
        return _EntropyFn.apply(x, kernel, bias, labels, ignore_index, reduction, scratch_limit)
    loss, rows, _, _, _ = _entropy(x, kernel, labels, bias, ignore_index, reduction, 1.0, scratch_limit, row_losses, (False, False, False), False)
    return (loss, rows.reshape(labels.shape)) if row_losses else loss
