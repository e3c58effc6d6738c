"""CPU: what axc_scale refuses before it looks for a device."""
import ctypes as C

from test_gpu_scale import Part


def test_refusals(built):
    from tf_approximate_b200 import _lib
    L = _lib.load()
    good = dict(x=256, out=512, count=4, type=1)
    factor, none = C.c_void_p(1024), C.c_void_p()
    assert L.axc_scale(None, 0, factor, 0, none) == 0 and L.axc_scale((Part * 1)(Part(None, None, 0, 0)), 1, factor, 0, none) == 0
    for change in ({"x": None}, {"out": None}, {"count": -1}, {"count": 1 << 50}, {"type": 3}, {"type": -1}, {"x": 257}, {"out": 513}, {"type": 0, "x": 258}):
        assert L.axc_scale((Part * 1)(Part(**{**good, **change})), 1, factor, 0, none) == 3, change
    assert L.axc_scale((Part * 1)(Part(**good)), 1, none, 0, none) == 3 and L.axc_scale((Part * 1)(Part(**good)), 1, C.c_void_p(1026), 0, none) == 3
    assert L.axc_scale(None, 1, factor, 0, none) == 3 and L.axc_scale((Part * 1)(Part(**good)), -1, factor, 0, none) == 3
