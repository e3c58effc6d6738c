"""GPU: calls with nothing to compute leave a status word of 0, whatever the workspace held before."""
import ctypes as C

import pytest

from test_dense_refusals import Dense
from test_gpu_dense_edges import pointer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,inputs,units", [(0, 8, 16), (5, 0, 16), (5, 8, 0), (0, 0, 16), (0, 8, 0), (5, 0, 0), (0, 0, 0), (5, 8, 16)])
@pytest.mark.parametrize("activation", [0, 1])
def test_status_of_empty_sizes(built, rows, inputs, units, dtype, activation):
    import torch
    from tf_approximate_b200 import _lib
    L, dt = _lib.load(), getattr(torch, dtype)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    x, w, y, b = (torch.ones(*s, device="cuda", dtype=dt) for s in ((rows, inputs), (inputs, units), (rows, units), (units,)))
    d = Dense(rows=rows, inputs=inputs, units=units, type=("float32", "bfloat16").index(dtype), bias_type=("float32", "bfloat16").index(dtype), activation=activation,
              transposed=0, xr=max(inputs, 1), xc=1, kr=max(units, 1), kc=1, rr=max(units, 1))
    sizes = (C.c_size_t(), C.c_size_t())
    assert L.axc_dense_workspace_bytes(C.byref(d), pointer(x), pointer(w), 0, C.byref(sizes[0]), C.byref(sizes[1])) == 0
    out = [torch.empty_like(t) for t in (x, w, b)]
    for backward in (False, True):
        ws = torch.full((max(256, sizes[backward].value),), 0xA5, dtype=torch.uint8, device="cuda")
        if backward:
            rc = L.axc_dense_backward(C.byref(d), pointer(y), pointer(x), pointer(w), pointer(y), *map(pointer, out), None, pointer(ws), sizes[1], 0, stream)
        else:
            rc = L.axc_dense_forward(C.byref(d), pointer(x), pointer(w), pointer(b), None, pointer(y.clone()), None, pointer(ws), sizes[0], 0, stream)
        word = C.c_int32(-1)
        assert rc == 0 and L.axc_matrix_status(pointer(ws), C.byref(word), 0, stream) == 0
        assert word.value == 0, (backward, hex(word.value & 0xffffffff))


def test_checked_calls_on_empty_sizes(built):
    """`check` asks for the status, whose memory the caching allocator hands out as it was left."""
    import torch
    import tf_approximate_b200 as ax
    for t, k, n in ((0, 8, 16), (5, 0, 16), (5, 8, 0), (0, 0, 0)):
        x, w, b = torch.ones(t, k, device="cuda"), torch.ones(k, n, device="cuda"), torch.ones(n, device="cuda")
        for size in (512, 1024, 2048, 4096):
            torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda")
        _, kept = ax.dense_forward(x, w, b, None, "relu", check=True)
        ax.dense_backward(torch.ones(t, n, device="cuda"), x, w, kept, "relu", bias=b, check=True)
