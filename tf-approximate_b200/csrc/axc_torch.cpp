// The way from torch tensors to the C entry points of the dense layer, the cross entropy and AdamW: checks, outputs, scratch and
// the call.  Written against CPython and ATen because a call of these operators takes 5 to 30 us on the GPU, and the same
// steps in Python took 15 to 100.  The entry points' addresses come from the loaded library (init), so that this module serves either
// flavour of it.  Every function translates C++ exceptions.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>

#include <string>
#include <vector>

#include "axconv.h"

namespace {

struct Entry {
    decltype(&axc_dense_workspace_bytes) dense_bytes;
    decltype(&axc_dense_forward) dense_forward;
    decltype(&axc_dense_backward) dense_backward;
    decltype(&axc_matrix_status) status;
    decltype(&axc_entropy_workspace_bytes) entropy_bytes;
    decltype(&axc_entropy) entropy;
    decltype(&axc_adamw_step) adamw;
    decltype(&axc_scale) scale;
};
Entry g_entry = {};
PyObject *g_invalid = nullptr, *g_internal = nullptr, *g_raise = nullptr;    // exception classes; raise_for_status(status, what)

// A Python exception is set: unwinds to the function's end.
struct Raised {};

[[noreturn]] void invalid(const std::string &text)
{
    PyErr_SetString(g_invalid, text.c_str());
    throw Raised();
}
void check(int status, const char *what)
{
    if (status == AXC_OK) return;
    PyObject *r = PyObject_CallFunction(g_raise, "is", status, what);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(g_internal, what);
    throw Raised();
}

#define AXC_TORCH_BEGIN \
    HANDLE_TH_ERRORS    \
    try {
#define AXC_TORCH_END                  \
    } catch (const Raised &) {         \
        return nullptr;                \
    }                                  \
    END_HANDLE_TH_ERRORS

int type_of(const at::Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return AXC_TYPE_FLOAT32;
    case at::kBFloat16: return AXC_TYPE_BFLOAT16;
    case at::kHalf: return AXC_TYPE_FLOAT16;
    default: return -1;
    }
}
std::string text_of(at::IntArrayRef shape)
{
    std::string s = "(";
    for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    return s + (shape.size() == 1 ? ",)" : ")");
}
// a tensor, or an undefined one for None
at::Tensor tensor_of(PyObject *o, const char *name, bool optional)
{
    if (o == Py_None && optional) return at::Tensor();
    if (!THPVariable_Check(o)) invalid(std::string(name) + " must be a torch tensor");
    const at::Tensor &t = THPVariable_Unpack(o);
    return t.is_neg() ? t.resolve_neg() : t;               // the imaginary part of a conjugate: its memory holds the other sign
}
PyObject *wrap(const at::Tensor &t)
{
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
const void *address(const at::Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out_address(const at::Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
void *stream_of(const at::Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

int64_t rows_of(at::IntArrayRef shape)
{
    int64_t n = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) n *= shape[i];
    return n;
}
at::Tensor as_rows(const at::Tensor &t)
{
    return t.dim() == 2 ? t : t.reshape({rows_of(t.sizes()), t.size(-1)});
}

struct Operands {
    at::Tensor x, kernel, bias;
    std::vector<int64_t> shape;                // of the output
    bool transposed;                           // the kernel lies in memory as [units, inputs]: its gradient then does too
    int device;
};

Operands operands(PyObject *px, PyObject *pk, PyObject *pb)
{
    Operands o;
    const at::Tensor x = tensor_of(px, "x", false);
    o.kernel = tensor_of(pk, "kernel", false);
    if (!x.is_cuda() || o.kernel.device() != x.device()) invalid("x and kernel must live on one CUDA device (this build has no CPU kernel)");
    if (type_of(x) < 0 || o.kernel.scalar_type() != x.scalar_type()) invalid("x and kernel must have one type, float32, bfloat16 or float16");
    if (x.dim() < 1 || o.kernel.dim() != 2 || o.kernel.size(0) != x.size(-1))
        invalid("x [..., inputs] and kernel [inputs, units] expected, got " + text_of(x.sizes()) + " and " + text_of(o.kernel.sizes()));
    const at::Tensor bias = tensor_of(pb, "bias", true);
    if (bias.defined()) {
        if (type_of(bias) < 0 || bias.device() != x.device() || bias.dim() != 1 || bias.size(0) != o.kernel.size(1))
            invalid("bias must be a float32, bfloat16 or float16 tensor of shape (" + std::to_string(o.kernel.size(1)) + ",) on x's device");
        o.bias = bias.contiguous();
    }
    o.shape.assign(x.sizes().begin(), x.sizes().end());
    o.shape.back() = o.kernel.size(1);
    o.x = as_rows(x);
    o.transposed = o.kernel.stride(0) == 1 && o.kernel.stride(1) != 1;
    o.device = x.device().index();
    return o;
}

// A tensor that goes with the output, as rows of `units` values
at::Tensor companion(PyObject *p, const char *name, const Operands &o)
{
    const at::Tensor t = tensor_of(p, name, false);
    if (t.scalar_type() != o.x.scalar_type() || t.device() != o.x.device() || t.sizes() != at::IntArrayRef(o.shape))
        invalid(std::string(name) + " must be a tensor of x's type, of shape " + text_of(o.shape) + " on x's device");
    return as_rows(t);
}

axc_dense_desc dense_desc(const Operands &o, int activation)
{
    axc_dense_desc d = {};
    d.rows = o.x.size(0);
    d.inputs = o.x.size(1);
    d.units = o.kernel.size(1);
    d.type = type_of(o.x);
    d.bias_type = o.bias.defined() ? type_of(o.bias) : AXC_TYPE_FLOAT32;
    d.activation = activation;
    d.kernel_gradient_transposed = o.transposed;
    d.x_row_stride = o.x.stride(0);
    d.x_column_stride = o.x.stride(1);
    d.kernel_row_stride = o.kernel.stride(0);
    d.kernel_column_stride = o.kernel.stride(1);
    return d;
}

at::Tensor scratch(const at::Tensor &like, size_t bytes) { return at::empty({int64_t(bytes)}, like.options().dtype(at::kByte)); }

void check_waits(const at::Tensor &ws, int device, void *stream)
{
    int32_t word = -1;
    check(g_entry.status(ws.const_data_ptr(), &word, device, stream), "status");
    if (word != 0) {
        PyErr_Format(g_internal, "a wait inside a matrix kernel ran out (status %d): the result is not valid", int(word));
        throw Raised();
    }
}

// dense_forward(x, kernel, bias, residual, activation, check) -> (y, kept)
PyObject *dense_forward(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    AXC_TORCH_BEGIN
    if (n != 6) invalid("dense_forward takes 6 arguments");
    c10::NoGradGuard no_grad;
    const Operands o = operands(a[0], a[1], a[2]);
    const int activation = int(PyLong_AsLong(a[4]));
    at::Tensor residual;
    axc_dense_desc d = dense_desc(o, activation);
    if (a[3] != Py_None) {
        residual = companion(a[3], "residual", o);
        if (residual.stride(1) != 1 && residual.size(1) > 1) residual = residual.contiguous();
        d.residual_row_stride = residual.stride(0);
    }
    const at::Tensor y = at::empty(o.shape, o.x.options());
    at::Tensor pre;
    if (activation == AXC_ACTIVATION_GELU || activation == AXC_ACTIVATION_SILU) {
        if (a[5] == Py_None) pre = at::Tensor();               // nobody asks for what the gradient needs
        else pre = at::empty(o.shape, o.x.options());
    }
    size_t bytes = 0;
    check(g_entry.dense_bytes(&d, address(o.x), address(o.kernel), o.device, &bytes, nullptr), "dense");
    const at::Tensor ws = scratch(o.x, bytes);
    void *stream = stream_of(o.x);
    check(g_entry.dense_forward(&d, address(o.x), address(o.kernel), address(o.bias), address(residual), out_address(y), out_address(pre), out_address(ws), bytes,
                                o.device, stream),
          "dense");
    if (a[5] == Py_True && y.numel()) check_waits(ws, o.device, stream);
    return Py_BuildValue("(NN)", wrap(y), activation == AXC_ACTIVATION_RELU ? wrap(y) : wrap(pre));
    AXC_TORCH_END
}

// dense_backward(grad, x, kernel, kept, activation, bias, residual, need_x, need_kernel, check) -> (dx, dkernel, dbias, dresidual)
PyObject *dense_backward(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    AXC_TORCH_BEGIN
    if (n != 10) invalid("dense_backward takes 10 arguments");
    c10::NoGradGuard no_grad;
    const Operands o = operands(a[1], a[2], a[5]);
    const int activation = int(PyLong_AsLong(a[4]));
    const at::Tensor grad = companion(a[0], "grad", o).contiguous();
    at::Tensor kept;
    if (activation != AXC_ACTIVATION_NONE) kept = companion(a[3], "kept", o).contiguous();
    const axc_dense_desc d = dense_desc(o, activation);
    at::Tensor dx, dkernel, dbias, dresidual;
    const at::TensorOptions options = o.x.options();
    if (a[7] == Py_True) {
        std::vector<int64_t> shape = o.shape;
        shape.back() = d.inputs;
        dx = at::empty(shape, options);
    }
    if (a[8] == Py_True) dkernel = o.transposed ? at::empty({d.units, d.inputs}, options) : at::empty({d.inputs, d.units}, options);
    if (o.bias.defined()) dbias = at::empty({d.units}, o.bias.options());
    const bool with_residual = a[6] != Py_None;
    if (with_residual) {
        companion(a[6], "residual", o);
        if (activation != AXC_ACTIVATION_NONE) dresidual = at::empty(o.shape, options);
    }
    size_t bytes = 0;
    check(g_entry.dense_bytes(&d, address(o.x), address(o.kernel), o.device, nullptr, &bytes), "dense gradients");
    const at::Tensor ws = scratch(o.x, bytes);
    void *stream = stream_of(o.x);
    check(g_entry.dense_backward(&d, address(grad), address(o.x), address(o.kernel), address(kept), out_address(dx), out_address(dkernel), out_address(dbias),
                                 out_address(dresidual), out_address(ws), bytes, o.device, stream),
          "dense gradients");
    if (a[9] == Py_True && (dx.defined() || dkernel.defined())) check_waits(ws, o.device, stream);
    if (dkernel.defined() && o.transposed) dkernel = dkernel.t();
    PyObject *r = nullptr;
    if (!with_residual) {
        Py_INCREF(Py_None);
        r = Py_None;
    } else if (activation == AXC_ACTIVATION_NONE) {            // its gradient is the output's
        Py_INCREF(a[0]);
        r = a[0];
    } else r = wrap(dresidual);
    return Py_BuildValue("(NNNN)", wrap(dx), wrap(dkernel), wrap(dbias), r);
    AXC_TORCH_END
}

// entropy(x, kernel, labels, bias, ignore_index, reduction, grad_scale, scratch_limit, row_losses, need_x, need_kernel, need_bias, check)
// -> (loss, rows, dx, dkernel, dbias)
PyObject *entropy(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    AXC_TORCH_BEGIN
    if (n != 13) invalid("entropy takes 13 arguments");
    c10::NoGradGuard no_grad;
    const Operands o = operands(a[0], a[1], a[3]);
    at::Tensor labels = tensor_of(a[2], "labels", false);
    const at::IntArrayRef lead(o.shape.data(), o.shape.size() - 1);
    if (labels.scalar_type() != at::kLong || labels.device() != o.x.device() || labels.sizes() != lead)
        invalid("labels must be an int64 tensor of shape " + text_of(lead) + " on x's device");
    if (o.kernel.size(0) == 0 || o.kernel.size(1) == 0) invalid("a classifier needs inputs and classes");
    labels = labels.contiguous();
    axc_entropy_desc d = {};
    d.rows = o.x.size(0);
    d.inputs = o.x.size(1);
    d.classes = o.kernel.size(1);
    d.type = type_of(o.x);
    d.bias_type = o.bias.defined() ? type_of(o.bias) : AXC_TYPE_FLOAT32;
    d.reduction = int(PyLong_AsLong(a[5]));
    d.kernel_gradient_transposed = o.transposed;
    d.ignore_index = PyLong_AsLongLong(a[4]);
    d.scratch_limit = PyLong_AsLongLong(a[7]);
    d.x_row_stride = o.x.stride(0);
    d.x_column_stride = o.x.stride(1);
    d.kernel_row_stride = o.kernel.stride(0);
    d.kernel_column_stride = o.kernel.stride(1);
    d.grad_scale = float(PyFloat_AsDouble(a[6]));
    if (PyErr_Occurred()) throw Raised();
    const at::TensorOptions options = o.x.options();
    const at::Tensor loss = at::empty({}, options.dtype(at::kFloat));
    at::Tensor rows, dx, dkernel, dbias;
    if (a[8] == Py_True) rows = at::empty(lead, options.dtype(at::kFloat));
    if (a[9] == Py_True) {
        std::vector<int64_t> shape = o.shape;
        shape.back() = d.inputs;
        dx = at::empty(shape, options);
    }
    if (a[10] == Py_True) dkernel = o.transposed ? at::empty({d.classes, d.inputs}, options) : at::empty({d.inputs, d.classes}, options);
    if (a[11] == Py_True && o.bias.defined()) dbias = at::empty({d.classes}, o.bias.options());
    const bool gradients = dx.defined() || dkernel.defined() || dbias.defined();
    size_t bytes = 0;
    check(g_entry.entropy_bytes(&d, address(o.x), address(o.kernel), o.device, gradients ? nullptr : &bytes, gradients ? &bytes : nullptr), "dense cross entropy");
    const at::Tensor ws = scratch(o.x, bytes);
    void *stream = stream_of(o.x);
    check(g_entry.entropy(&d, address(o.x), address(o.kernel), address(o.bias), labels.const_data_ptr<int64_t>(), static_cast<float *>(out_address(loss)),
                          static_cast<float *>(out_address(rows)), out_address(dx), out_address(dkernel), out_address(dbias), out_address(ws), bytes, o.device, stream),
          "dense cross entropy");
    if (a[12] == Py_True) check_waits(ws, o.device, stream);
    if (dkernel.defined() && o.transposed) dkernel = dkernel.t();
    return Py_BuildValue("(NNNNN)", wrap(loss), wrap(rows), wrap(dx), wrap(dkernel), wrap(dbias));
    AXC_TORCH_END
}

// scaled(factor, tensor or None, ...) -> a tuple of their products with the factor, a tensor of one value; tensors without gaps
PyObject *scaled(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    AXC_TORCH_BEGIN
    if (n < 1) invalid("scaled takes a factor");
    c10::NoGradGuard no_grad;
    at::Tensor factor = tensor_of(a[0], "factor", false);
    if (!factor.is_cuda() || factor.numel() != 1) invalid("the factor must be one value on a CUDA device");
    if (factor.scalar_type() != at::kFloat) factor = factor.to(at::kFloat);
    std::vector<at::Tensor> x(n - 1), out(n - 1);
    std::vector<axc_scale_tensor> table;
    for (Py_ssize_t i = 0; i + 1 < n; ++i) {
        x[i] = tensor_of(a[i + 1], "tensor", true);
        if (!x[i].defined()) continue;
        if (type_of(x[i]) < 0 || x[i].device() != factor.device()) invalid("a float32, bfloat16 or float16 tensor on the factor's device expected");
        if (!x[i].is_non_overlapping_and_dense()) x[i] = x[i].contiguous();
        out[i] = at::empty_like(x[i]);
        if (out[i].strides() != x[i].strides()) x[i] = x[i].contiguous(), out[i] = at::empty_like(x[i], at::MemoryFormat::Contiguous);
        table.push_back({address(x[i]), out_address(out[i]), x[i].numel(), type_of(x[i])});
    }
    check(g_entry.scale(table.data(), int32_t(table.size()), static_cast<const float *>(address(factor)), factor.device().index(), stream_of(factor)), "scale");
    PyObject *r = PyTuple_New(n - 1);
    if (!r) throw Raised();
    for (Py_ssize_t i = 0; i + 1 < n; ++i) PyTuple_SET_ITEM(r, i, wrap(out[i]));
    return r;
    AXC_TORCH_END
}

// adamw_step(params, grads or None, the table's address, exp_avg, type, state_bits, step, (beta1, beta2, eps, grad_scale), exp_avg_sq, its scales)
// params and grads: lists; the table's entries have counts and rates already.
PyObject *adamw_step(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    AXC_TORCH_BEGIN
    if (n != 11 || !PyList_Check(a[0]) || (a[1] != Py_None && !PyList_Check(a[1]))) invalid("adamw_step takes 11 arguments");
    c10::NoGradGuard no_grad;
    axc_adamw_tensor *table = static_cast<axc_adamw_tensor *>(PyLong_AsVoidPtr(a[2]));
    const int type = int(PyLong_AsLong(a[4]));
    axc_adamw_desc d = {};
    d.type = type;
    d.state_bits = int(PyLong_AsLong(a[5]));
    d.step = PyLong_AsLongLong(a[6]);
    if (!PyArg_ParseTuple(a[7], "dddf", &d.beta1, &d.beta2, &d.eps, &d.grad_scale)) throw Raised();
    const at::Tensor m = tensor_of(a[3], "moments", false), v = tensor_of(a[8], "moments", false), ms = tensor_of(a[9], "scales", true),
                     vs = tensor_of(a[10], "scales", true);
    if (PyErr_Occurred()) throw Raised();
    const Py_ssize_t count = PyList_GET_SIZE(a[0]);
    const bool given = a[1] != Py_None;
    if (given && PyList_GET_SIZE(a[1]) != count)
        invalid(std::to_string(PyList_GET_SIZE(a[1])) + " gradients for " + std::to_string(count) + " parameters");
    const int device = m.device().index();                                // the parameters'
    std::vector<at::Tensor> copies;
    auto fits = [&](const at::Tensor &t, const char *what) {
        if (!t.is_cuda() || t.device().index() != device || type_of(t) != type) invalid(std::string("every ") + what + " must be a tensor of the optimizer's type and device");
    };
    // the moments are attributes that a caller can replace: they are what the kernels take them for, or nothing is launched
    int64_t blocks = 0;
    for (Py_ssize_t i = 0; i < count; ++i) blocks += table[i].count / AXC_ADAMW_BLOCK + (table[i].count % AXC_ADAMW_BLOCK != 0);
    auto holds = [&](const at::Tensor &t, int64_t values, at::ScalarType scalar) {
        if (!t.defined() || !t.is_cuda() || t.device().index() != device || t.scalar_type() != scalar || t.numel() != values || !t.is_contiguous())
            invalid("the optimizer's moments are not the tensors that it made");
    };
    const at::ScalarType state = d.state_bits == 8 ? at::kFloat8_e4m3fn : at::kFloat;
    holds(m, blocks * AXC_ADAMW_BLOCK, state);
    holds(v, blocks * AXC_ADAMW_BLOCK, state);
    if (d.state_bits == 8) {
        holds(ms, blocks, at::kFloat);
        holds(vs, blocks, at::kFloat);
    }
    d.exp_avg = out_address(m);
    d.exp_avg_sq = out_address(v);
    d.exp_avg_scale = static_cast<float *>(out_address(ms));
    d.exp_avg_sq_scale = static_cast<float *>(out_address(vs));
    // (by reference: copies of 161 tensors cost a microsecond)
    for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject *const item = PyList_GET_ITEM(a[0], i);
        if (!THPVariable_Check(item)) invalid("parameter must be a torch tensor");
        const at::Tensor &p = THPVariable_Unpack(item);
        fits(p, "parameter");
        if (p.numel() != table[i].count) invalid("a parameter has another size than it had when the optimizer was made");
        if (!p.is_contiguous()) invalid("parameters must be contiguous");
        if (p.is_neg()) invalid("a parameter whose memory holds the other sign");
        table[i].param = p.mutable_data_ptr();
        table[i].grad = nullptr;
        PyObject *const gradient = given ? PyList_GET_ITEM(a[1], i) : nullptr;
        if (gradient == Py_None) continue;
        if (gradient && !THPVariable_Check(gradient)) invalid("gradient must be a torch tensor");
        const at::Tensor &g = gradient ? THPVariable_Unpack(gradient) : p.grad();
        if (!g.defined()) continue;
        fits(g, "gradient");
        if (g.sizes() != p.sizes()) invalid("a gradient has another shape than its parameter: " + text_of(g.sizes()) + " for " + text_of(p.sizes()));
        if (g.is_contiguous() && !g.is_neg()) table[i].grad = g.const_data_ptr();
        else {
            copies.push_back(g.resolve_neg().contiguous());
            table[i].grad = copies.back().const_data_ptr();
        }
    }
    check(g_entry.adamw(&d, table, int32_t(count), device, stream_of(m)), "AdamW");
    // a graph that saved a parameter's value from before the step is refused its backward pass
    for (Py_ssize_t i = 0; i < count; ++i) {
        const at::Tensor &p = THPVariable_Unpack(PyList_GET_ITEM(a[0], i));
        if (table[i].grad && !p.is_inference()) p.unsafeGetTensorImpl()->bump_version();        // (tensors of inference mode have no counter)
    }
    Py_RETURN_NONE;
    AXC_TORCH_END
}

// init(addresses of the entry points, InvalidArgumentError, InternalError, raise_for_status)
PyObject *init(PyObject *, PyObject *args)
{
    unsigned long long p[8];
    PyObject *i, *e, *r;
    if (!PyArg_ParseTuple(args, "(KKKKKKKK)OOO", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6], &p[7], &i, &e, &r)) return nullptr;
    g_entry.dense_bytes = reinterpret_cast<decltype(g_entry.dense_bytes)>(p[0]);
    g_entry.dense_forward = reinterpret_cast<decltype(g_entry.dense_forward)>(p[1]);
    g_entry.dense_backward = reinterpret_cast<decltype(g_entry.dense_backward)>(p[2]);
    g_entry.status = reinterpret_cast<decltype(g_entry.status)>(p[3]);
    g_entry.entropy_bytes = reinterpret_cast<decltype(g_entry.entropy_bytes)>(p[4]);
    g_entry.entropy = reinterpret_cast<decltype(g_entry.entropy)>(p[5]);
    g_entry.adamw = reinterpret_cast<decltype(g_entry.adamw)>(p[6]);
    g_entry.scale = reinterpret_cast<decltype(g_entry.scale)>(p[7]);
    Py_INCREF(i);
    Py_INCREF(e);
    Py_INCREF(r);
    g_invalid = i;
    g_internal = e;
    g_raise = r;
    Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {{"init", init, METH_VARARGS, nullptr},
                           {"dense_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dense_forward)), METH_FASTCALL, nullptr},
                           {"dense_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dense_backward)), METH_FASTCALL, nullptr},
                           {"entropy", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entropy)), METH_FASTCALL, nullptr},
                           {"scaled", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scaled)), METH_FASTCALL, nullptr},
                           {"adamw_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw_step)), METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_axc_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__axc_torch() { return PyModule_Create(&g_module); }
