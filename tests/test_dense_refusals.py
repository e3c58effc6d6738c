"""CPU: what the C entry points of the dense layer, the cross entropy and AdamW refuse before they touch a GPU, and what the Python
functions refuse without one."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def L(built):
    from tf_approximate_b200 import _lib
    return _lib.load()


class Dense(C.Structure):
    _fields_ = ([(n, C.c_int64) for n in ("rows", "inputs", "units")] + [(n, C.c_int32) for n in ("type", "bias_type", "activation", "transposed")] +
                [(n, C.c_int64) for n in ("xr", "xc", "kr", "kc", "rr")])


class Entropy(C.Structure):
    _fields_ = ([(n, C.c_int64) for n in ("rows", "inputs", "classes")] + [(n, C.c_int32) for n in ("type", "bias_type", "reduction", "transposed")] +
                [(n, C.c_int64) for n in ("ignore", "limit", "xr", "xc", "kr", "kc")] + [("scale", C.c_float)])


class Adamw(C.Structure):
    _fields_ = [("type", C.c_int32), ("bits", C.c_int32), ("step", C.c_int64), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double),
                ("scale", C.c_float), ("m", C.c_void_p), ("v", C.c_void_p), ("ms", C.c_void_p), ("vs", C.c_void_p)]


class Tensor(C.Structure):
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("count", C.c_int64), ("lr", C.c_double), ("decay", C.c_double)]


def test_dense_descriptions(L):
    good = dict(rows=4, inputs=8, units=16, type=1, bias_type=0, activation=1, transposed=0, xr=8, xc=1, kr=16, kc=1, rr=16)
    for name, value in (("rows", -1), ("inputs", -1), ("units", 1 << 40), ("type", 3), ("bias_type", -1), ("activation", 4), ("xr", -8), ("kc", -1)):
        d = Dense(**{**good, name: value})
        assert L.axc_dense_workspace_bytes(C.byref(d), None, None, 0, None, None) == 3, name
    d = Dense(**good)
    assert L.axc_dense_workspace_bytes(None, None, None, 0, None, None) == 3
    null = [C.c_void_p()] * 4
    # no output, no operands: refused before a device is looked for; nothing to do: fine
    assert L.axc_dense_forward(C.byref(d), *null, C.c_void_p(), C.c_void_p(), C.c_void_p(), C.c_size_t(0), 0, C.c_void_p()) == 3
    d = Dense(**{**good, "rows": 0})
    assert L.axc_dense_forward(C.byref(d), *null, C.c_void_p(), C.c_void_p(), C.c_void_p(), C.c_size_t(0), 0, C.c_void_p()) == 0
    d = Dense(**good)
    assert L.axc_dense_backward(C.byref(d), *null, *null, C.c_void_p(), C.c_size_t(0), 0, C.c_void_p()) == 3
    assert L.axc_matrix_status(None, None, 0, None) == 3


def test_entropy_descriptions(L):
    good = dict(rows=4, inputs=8, classes=16, type=1, bias_type=0, reduction=0, transposed=0, ignore=-100, limit=0, xr=8, xc=1, kr=16, kc=1, scale=1.0)
    for name, value in (("rows", -1), ("inputs", 0), ("classes", 0), ("type", 5), ("reduction", 2), ("kr", -1)):
        d = Entropy(**{**good, name: value})
        assert L.axc_entropy_workspace_bytes(C.byref(d), None, None, 0, None, None) == 3, name
    d = Entropy(**good)
    assert L.axc_entropy(C.byref(d), *[C.c_void_p()] * 10, C.c_size_t(0), 0, C.c_void_p()) == 3


def test_adamw_descriptions(L):
    blocks = C.c_int64()
    counts = (C.c_int64 * 4)(0, 1, 256, 257)
    assert L.axc_adamw_state_blocks(counts, 4, C.byref(blocks)) == 0 and blocks.value == 4
    assert L.axc_adamw_state_blocks((C.c_int64 * 1)(-1), 1, C.byref(blocks)) == 3
    assert L.axc_adamw_state_blocks((C.c_int64 * 1)(1 << 60), 1, C.byref(blocks)) == 3
    good = dict(type=0, bits=8, step=1, beta1=0.9, beta2=0.999, eps=1e-8, scale=1.0, m=256, v=512, ms=1024, vs=2048)
    one = Tensor(256, 512, 4, 1e-3, 0.0)
    for name, value in (("type", 3), ("bits", 16), ("step", 0), ("beta1", 1.0), ("beta2", -0.1), ("eps", -1.0), ("m", None), ("v", 257), ("ms", None)):
        assert L.axc_adamw_step(C.byref(Adamw(**{**good, name: value})), C.byref(one), 1, 0, C.c_void_p()) == 3, name
    for t in (Tensor(None, 512, 4, 1e-3, 0.0), Tensor(258, 512, 4, 1e-3, 0.0), Tensor(256, 512, -1, 1e-3, 0.0)):
        assert L.axc_adamw_step(C.byref(Adamw(**good)), C.byref(t), 1, 0, C.c_void_p()) == 3
    assert L.axc_adamw_step(C.byref(Adamw(**good)), None, 0, 0, C.c_void_p()) == 0


def test_python_refusals_without_a_gpu(built):
    import torch
    import tf_approximate_b200 as ax
    x, w = torch.zeros(2, 3), torch.zeros(3, 4)
    for call in (lambda: ax.dense(x, w), lambda: ax.dense(None, w), lambda: ax.dense(x, w, activation="tanh"), lambda: ax.dense_backward(x, x, w),
                 lambda: ax.dense_cross_entropy(x, w, torch.zeros(2, dtype=torch.int64)), lambda: ax.dense_cross_entropy(x, w, x, reduction="none"),
                 lambda: ax.AdamW([x]), lambda: ax.AdamW([]), lambda: ax.Dense(3, 4, activation="tanh")):
        with pytest.raises(ax.InvalidArgumentError):
            call()
