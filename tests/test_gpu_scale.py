"""GPU: tensors times one fp32 factor in device memory, rounded once, through the C entry point and the module between torch and it."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


class Part(C.Structure):
    _fields_ = [("x", C.c_void_p), ("out", C.c_void_p), ("count", C.c_int64), ("type", C.c_int32)]


@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("factor", [1.0 / 3.0, 65536.0, 0.0, float("inf")])
def test_every_value_is_rounded_once(built, factor, offset):
    import torch
    from tf_approximate_b200 import _lib
    g = torch.Generator(device="cuda").manual_seed(offset)
    types = (torch.float32, torch.bfloat16, torch.float16)
    sizes = [0, 1, 7, 4095, 4096, 4097, 8192, 8193, 100003, 3]
    dtypes = [types[i % 3] for i in range(len(sizes))]
    x = [torch.randn(n + 16, device="cuda", generator=g).to(t) for n, t in zip(sizes, dtypes)]
    out = [torch.full((n + 16,), 77.0, device="cuda", dtype=t) for n, t in zip(sizes, dtypes)]
    parts = (Part * len(sizes))(*[Part(a[offset:].data_ptr(), b[offset:].data_ptr(), n, types.index(t)) for a, b, n, t in zip(x, out, sizes, dtypes)])
    f = torch.tensor([factor], device="cuda")
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert _lib.load().axc_scale(parts, len(sizes), C.c_void_p(f.data_ptr()), 0, stream) == 0
    for a, b, n in zip(x, out, sizes):
        want = (a.float() * f).to(a.dtype)[offset:offset + n]
        got = b[offset:offset + n]
        assert torch.equal(torch.nan_to_num(got, 5.0, 6.0, 7.0), torch.nan_to_num(want, 5.0, 6.0, 7.0))
        assert bool((b[:offset] == 77).all()) and bool((b[offset + n:] == 77).all())


def test_memory_order_is_kept(built):
    import torch
    from tf_approximate_b200 import _lib
    f = torch.tensor(0.25, device="cuda")
    a, b = torch.randn(30, 40, device="cuda").t(), torch.randn(20, 30, device="cuda", dtype=torch.bfloat16)[:, ::2]
    got = _lib.binding().scaled(f, a, None, b, torch.zeros(0, 4, device="cuda"))
    assert torch.equal(got[0], a * 0.25) and got[0].stride() == a.stride() and got[1] is None
    assert torch.equal(got[2], b * 0.25) and got[3].shape == (0, 4)
