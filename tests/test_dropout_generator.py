"""CPU: the generator that the tests of dropout compare with, against the answers that its authors publish, and its two forms against each other;
what the C entry points of dropout, group norm and the 8-bit dense layer refuse before they touch a GPU."""
import ctypes as C

import numpy as np
import pytest

import philox


def test_known_answers():
    for counter, key, want in (((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
                               ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
                               ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))):
        assert tuple(philox.words(counter, key)) == want


def test_both_forms_agree():
    seed, offset, first = 0x0123456789abcdef, 0xfedcba9876543210, 8 * (2 ** 33 + 5)
    got = philox.bits(first, 24, seed, offset)
    for i in range(24):
        j = (first + i) // 8
        w = philox.words((j & 0xffffffff, j >> 32, offset & 0xffffffff, offset >> 32), (seed & 0xffffffff, seed >> 32))[i % 8 // 2]
        assert got[i] == (w >> 16 if i % 2 else w & 0xffff)


class Dropout(C.Structure):
    _fields_ = [("count", C.c_int64), ("type", C.c_int32), ("rate", C.c_double), ("seed", C.c_uint64), ("offset", C.c_uint64)]


def test_descriptions(built):
    from tf_approximate_b200 import _lib
    L, null = _lib.load(), C.c_void_p()
    call = lambda x=256, y=512, r=None, o=None, device=0, **k: L.axc_dropout(  # noqa: E731
        C.byref(Dropout(**{**dict(count=8, type=1, rate=0.5, seed=1, offset=2), **k})), C.c_void_p(x), C.c_void_p(r), C.c_void_p(y), C.c_void_p(o), device, null)
    for bad in (dict(count=-1), dict(type=3), dict(type=-1), dict(rate=-0.1), dict(rate=1.5), dict(rate=float("nan")), dict(x=None), dict(y=None), dict(x=257), dict(y=513), dict(r=255),
                dict(o=260), dict(device=-1)):
        assert call(**bad) == 3, bad
    assert L.axc_dropout(None, null, null, null, null, 0, null) == 3
    assert call(count=0, x=None, y=None) == 0


class Norm(C.Structure):
    _fields_ = [(n, C.c_int64) for n in ("samples", "places", "channels", "groups")] + [(n, C.c_int32) for n in ("type", "scale", "offset", "act")] + [("eps", C.c_float)]


def test_group_norm_descriptions(built):
    from tf_approximate_b200 import _lib
    L, null, at = _lib.load(), C.c_void_p(), C.c_void_p
    good = dict(samples=2, places=9, channels=24, groups=6, type=1, scale=0, offset=0, act=3, eps=1e-3)
    for bad in (dict(samples=-1), dict(places=-1), dict(channels=0), dict(channels=25), dict(groups=0), dict(groups=-6), dict(type=3), dict(scale=-1), dict(offset=7), dict(act=4),
                dict(eps=-1.0), dict(eps=float("inf")), dict(eps=float("nan")), dict(samples=1 << 30, places=1 << 30), dict(channels=6 << 40)):
        d = Norm(**{**good, **bad})
        assert L.axc_group_norm_workspace_bytes(C.byref(d), 0, None, None) == 3, bad
        assert L.axc_group_norm_forward(C.byref(d), at(256), null, null, null, at(512), at(1024), null, C.c_size_t(0), 0, null) == 3, bad
    d = Norm(**good)
    forward = lambda x=256, y=512, s=1024, scale=None, res=None: L.axc_group_norm_forward(  # noqa: E731
        C.byref(d), at(x), at(scale), null, at(res), at(y), at(s), null, C.c_size_t(0), 0, null)
    for bad in (dict(x=None), dict(y=None), dict(s=None), dict(x=257), dict(y=513), dict(s=1028), dict(scale=258), dict(res=255)):
        assert forward(**bad) == 3, bad
    assert L.axc_group_norm_backward(C.byref(d), *[null] * 10, null, C.c_size_t(0), 0, null) == 3
    d = Norm(**{**good, "samples": 0})
    assert L.axc_group_norm_forward(C.byref(d), *[null] * 6, null, C.c_size_t(0), 0, null) == 0
    assert L.axc_group_norm_backward(C.byref(d), *[null] * 10, null, C.c_size_t(0), 0, null) == 0


class Dense8(C.Structure):
    _fields_ = [(n, C.c_int64) for n in ("rows", "inputs", "units")] + [(n, C.c_int32) for n in ("type", "bias", "act", "reserved")] + [(n, C.c_int64) for n in ("xr", "kr", "rr")]


def test_8bit_descriptions(built):
    from tf_approximate_b200 import _lib
    L, null, at = _lib.load(), C.c_void_p(), C.c_void_p
    good = dict(rows=40, inputs=200, units=300, type=1, bias=0, act=1, reserved=0, xr=200, kr=208, rr=300)
    for bad in (dict(rows=-1), dict(inputs=0), dict(units=-1), dict(units=1 << 40), dict(type=3), dict(bias=-1), dict(act=4), dict(xr=-1), dict(kr=-1), dict(rr=-1)):
        d, size = Dense8(**{**good, **bad}), C.c_size_t()
        assert L.axc_dense8_workspace_bytes(C.byref(d), null, 0, C.byref(size)) == 3, bad
        assert L.axc_dense8_forward(C.byref(d), at(256), at(512), at(768), null, null, at(1024), at(2048), C.c_size_t(1 << 30), 0, null) == 3, bad
    d = Dense8(**good)
    call = lambda x=256, k=512, s=768, b=None, r=None, y=1024: L.axc_dense8_forward(  # noqa: E731
        C.byref(d), at(x), at(k), at(s), at(b), at(r), at(y), null, C.c_size_t(0), 0, null)
    for bad in (dict(x=None), dict(k=None), dict(s=None), dict(y=None), dict(x=257), dict(s=770), dict(b=258), dict(r=255), dict(y=1025)):
        assert call(**bad) == 3, bad
    d = Dense8(**{**good, "rows": 0})
    assert call(x=None, y=None) == 0
    quantize = lambda x=256, rows=4, inputs=200, stride=200, type=1, block=1, codes=512, scales=1024, device=0: L.axc_quantize_blocks(  # noqa: E731
        at(x), C.c_int64(rows), C.c_int64(inputs), C.c_int64(stride), type, block, at(codes), at(scales), device, null)
    for bad in (dict(x=None), dict(codes=None), dict(scales=None), dict(rows=-1), dict(inputs=-1), dict(stride=-1), dict(type=5), dict(block=2), dict(x=257), dict(scales=1026), dict(device=-1),
                dict(rows=1 << 40)):
        assert quantize(**bad) == 3, bad
    assert quantize(rows=0, x=None) == 0


def test_python_refusals_without_a_gpu(built):
    import torch
    import tf_approximate_b200 as ax
    x = torch.zeros(2, 8)
    for call in (lambda: ax.dropout(x, 0.5, 1), lambda: ax.dropout(None, 0.5, 1), lambda: ax.group_norm(x, 2), lambda: ax.group_norm(None, 2), lambda: ax.quantize_blocks(x), lambda: ax.dense_8bit(x, x, x), lambda: ax.Dense8bit(None), lambda: ax.GroupNorm(8, 3),
                 lambda: ax.Dropout(1.5), lambda: ax.Dropout(-0.5), lambda: ax.GroupNorm(8, 0)):
        with pytest.raises(ax.InvalidArgumentError):
            call()
    assert ax.Dropout(0.5).eval()(x) is x
