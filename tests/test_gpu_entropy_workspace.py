"""GPU: the cross entropy's C entry point stays inside a workspace of exactly the size that it asks for, with classes just below a multiple
of 256 and pieces of unequal size, and its bias gradient is right there."""
import ctypes as C

import pytest

from test_dense_refusals import Entropy
from test_gpu_dense_edges import pointer
from test_gpu_dense_entropy import check_entropy, make

pytestmark = pytest.mark.gpu


# rows, classes, classes at a time (None: the exponentials are kept)
SIZES = [(4096, 5119, None), (2048, 10235, 5120), (2048, 9663, 4864), (2100, 4850, None)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,classes,piece", SIZES)
def test_workspace_has_room_for_the_sums_of_the_bias(built, rows, classes, piece, dtype):
    import torch
    from tf_approximate_b200 import _lib
    L = _lib.load()
    x, w, b, labels = make(rows, 64, classes, dtype, "in_out")
    limit = 0 if piece is None else rows * piece * (6 if dtype == "float32" else 2)
    d = Entropy(rows=rows, inputs=64, classes=classes, type=("float32", "bfloat16", "float16").index(dtype), bias_type=("float32", "bfloat16", "float16").index(dtype),
                reduction=0, transposed=0, ignore=-100, limit=limit, xr=64, xc=1, kr=classes, kc=1, scale=1.0)
    size = C.c_size_t()
    assert L.axc_entropy_workspace_bytes(C.byref(d), pointer(x), pointer(w), 0, None, C.byref(size)) == 0
    ws = torch.full((size.value + (1 << 18),), 0xA5, dtype=torch.uint8, device="cuda")
    loss, dx, dw, db = torch.empty((), device="cuda"), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    assert L.axc_entropy(C.byref(d), pointer(x), pointer(w), pointer(b), pointer(labels), pointer(loss), None, pointer(dx), pointer(dw), pointer(db),
                         pointer(ws), size, 0, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    assert bool((ws[size.value:] == 0xA5).all())
    check_entropy(x, w, b, labels, dtype, limit=limit or None, scale=256.0 if dtype == "float16" else 1.0)
