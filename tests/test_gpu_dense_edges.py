"""GPU: the dense layer's C entry points write nothing outside their buffers and depend on nothing outside their inputs: tensors that lie
in the middle of one allocation, with guard values and NaNs around them."""
import ctypes as C

import pytest

from test_dense_refusals import Dense

pytestmark = pytest.mark.gpu

GUARD = 64                       # values on either side: 256 bytes, so that a tensor's own alignment stays 16 bytes


class Arena:
    """One allocation of fp32 values, all `fill`; tensors are cut out of it with guards between them."""

    def __init__(self, values, fill):
        import torch
        self.all = torch.full((values,), fill, device="cuda")
        self.at, self.parts = 0, []

    def take(self, *shape, like=None):
        n = 1
        for s in shape:
            n *= s
        begin = self.at + GUARD
        self.at = begin + -(-n // 4) * 4
        assert self.at + GUARD <= self.all.numel()
        t = self.all[begin:begin + n].view(*shape)
        self.parts.append((begin, begin + n))
        if like is not None:
            t.copy_(like)
        return t

    def untouched(self):
        import torch
        keep = torch.ones(self.all.numel(), dtype=torch.bool, device="cuda")
        for a, b in self.parts:
            keep[a:b] = False
        return self.all[keep]


def pointer(t):
    return C.c_void_p(t.data_ptr() if t is not None else None)


@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("rows", [32, 96])
@pytest.mark.parametrize("units", [4, 12, 20, 100, 260])
def test_backward_stays_inside_its_buffers(built, units, rows, activation):
    """fp32 lines of a whole number of 16-byte groups, but not of two: the operand's lines are longer than the tensors'."""
    import torch
    import tf_approximate_b200 as ax
    from tf_approximate_b200 import _lib
    inputs, act = 24, ("none", "relu", "gelu", "silu").index(activation)
    g = torch.Generator(device="cuda").manual_seed(units + rows)
    x, w, b, r, dy = (torch.randn(*s, device="cuda", generator=g) for s in ((rows, inputs), (inputs, units), (units,), (rows, units), (rows, units)))
    _, kept = ax.dense_forward(x, w, b, r, activation)
    want = ax.dense_backward(dy, x, w, kept, activation, bias=b, residual=r)
    source, result = Arena(1 << 18, float("nan")), Arena(1 << 18, 12345.0)
    dy2 = source.take(rows, units, like=dy)
    kept2 = source.take(rows, units, like=kept) if kept is not None else None
    dr, dx, dw, db = result.take(rows, units), result.take(rows, inputs), result.take(inputs, units), result.take(units)
    d = Dense(rows=rows, inputs=inputs, units=units, type=0, bias_type=0, activation=act, transposed=0, xr=inputs, xc=1, kr=units, kc=1, rr=units)
    size = C.c_size_t()
    L = _lib.load()
    assert L.axc_dense_workspace_bytes(C.byref(d), pointer(x), pointer(w), 0, None, C.byref(size)) == 0
    ws = torch.full((size.value + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    assert L.axc_dense_backward(C.byref(d), pointer(dy2), pointer(x), pointer(w), pointer(kept2), pointer(dx), pointer(dw), pointer(db), pointer(dr),
                                pointer(ws), size, 0, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    assert bool((result.untouched() == 12345.0).all()) and bool((ws[size.value:] == 0xA5).all())
    assert bool(torch.isnan(source.untouched()).all())
    for got, expected in zip((dx, dw, db, dr), want):
        assert torch.equal(got, expected)
