"""CPU: the C entry points of the dense layer and the cross entropy refuse addresses that are not multiples of their type's size, before
they look for a device: a kernel would fault there."""
import ctypes as C

import pytest

from test_dense_refusals import Dense, Entropy


@pytest.fixture(scope="module")
def L(built):
    from tf_approximate_b200 import _lib
    return _lib.load()


@pytest.mark.parametrize("kind,size", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("bias_kind,bias_size", [(0, 4), (1, 2)])
def test_addresses_off_their_type(L, kind, size, bias_kind, bias_size):
    d = Dense(rows=4, inputs=8, units=16, type=kind, bias_type=bias_kind, activation=1, transposed=0, xr=8, xc=1, kr=16, kc=1, rr=16)
    e = Entropy(rows=4, inputs=8, classes=16, type=kind, bias_type=bias_kind, reduction=0, transposed=0, ignore=-100, limit=0, xr=8, xc=1, kr=16, kc=1, scale=1.0)
    tail = (C.c_void_p(), C.c_size_t(0), 0, C.c_void_p())
    cases = ((L.axc_dense_forward, d, (size, size, bias_size, size, size, size)), (L.axc_dense_backward, d, (size,) * 6 + (bias_size, size)),
             (L.axc_entropy, e, (size, size, bias_size, 8, 4, 4, size, size, bias_size)))
    for entry, desc, sizes in cases:
        good = [4096 * (i + 1) for i in range(len(sizes))]
        # no workspace, no device: anything but the refusal of an argument
        assert entry(C.byref(desc), *map(C.c_void_p, good), *tail) in (13, 100)
        for i, unit in enumerate(sizes):
            for off in (1, unit // 2):
                bad = list(good)
                bad[i] += off
                assert entry(C.byref(desc), *map(C.c_void_p, bad), *tail) == 3, (entry.__name__, i, off)
