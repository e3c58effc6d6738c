"""GPU: the dense layer, the cross entropy and AdamW in the debug flavour (libaxconv_check.so), in which every global index and every
shared-memory address of their kernels is checked before use.  A child process runs sizes and layouts that reach every kernel (tiles by pairs and
by lone CTAs, split sums, operands copied and read in place, few rows, packed and single values, few logits, kept exponentials, pieces of the
classes, whole and partial blocks of moments) against 64 bits, with the bounds of the operators' own tests, and must end with an empty violation record."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r"""
import ctypes as C, sys
import torch
sys.path[:0] = [%r, %r]
import tf_approximate_b200 as ax
from tf_approximate_b200 import _lib
L = _lib.load()
rec = (C.c_uint32 * 4)()
assert L.axc_debug_bounds_record(0, rec) == 0, "not the debug flavour"
g = torch.Generator(device="cuda").manual_seed(1)
from test_gpu_dense import check_dense
from test_gpu_dense_entropy import check_entropy

def clear(what):
    assert L.axc_debug_bounds_record(0, rec) == 0
    assert rec[0] == 0, (what, rec[0], "site", rec[1], "value", rec[2] | (rec[3] << 32))

def dense(x, w, b, r, act, dy):
    check_dense(x, w, b, r, act, str(dy.dtype)[6:], dy)
    clear(("dense", x.shape, w.shape, x.dtype, act))

for dtype in (torch.float32, torch.bfloat16, torch.float16):
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
    for t, k, n, act in ((33, 300, 136, "relu"), (64, 24, 260, "silu"), (1, 520, 1000, "silu"), (2, 4100, 72, None), (5, 31, 260, None), (8, 264, 3000, "gelu"),
                         (130, 72, 1000, "gelu"), (2100, 136, 4500, None), (300, 4096, 200, "silu"), (129, 65, 127, "relu"), (600, 200, 12, "gelu"), (17, 7, 20, "relu")):
        for order in range(2):
            w = rand(k, n) if order == 0 else rand(n, k).t()
            dense(rand(t, k), w, rand(n), rand(t, n) if (t + order) %% 2 else None, act, rand(t, n))
    # strides and starts of every kind
    t, k, n = 130, 72, 136
    for x, w, r in ((rand(k, t).t(), rand(k, n + 8)[:, 8:], rand(t, n + 4)[:, 4:]), (rand(t, k + 5)[:, 3:3 + k], rand(k, n + 1)[:, 1:], rand(n, t).t()),
                    (rand(t, 2 * k)[:, ::2], rand(n, k + 3)[:, :k].t(), rand(1, n).expand(t, n)), (rand(1, k).expand(t, k), rand(k, 1).expand(k, n), None),
                    (rand(t * k + 1)[1:].view(t, k), rand(2 * k, n)[::2], rand(t * n + 1)[1:].view(t, n))):
        dense(x, w, rand(n), r, "gelu", rand(t, n))
        dense(x[:2], w, rand(n), None, None, rand(2, n))
    # the last: the bias's partial sums at classes just below a multiple of 256
    for t, k, v, limit in ((100, 64, 300, None), (77, 40, 8192, None), (1600, 40, 900, None), (300, 64, 900, 1), (515, 65, 4099, 1 << 20), (1, 8, 10, None), (4096, 64, 5119, None),
                           (2048, 64, 10235, 2048 * 5120 * (6 if dtype == torch.float32 else 2))):
        for order in range(2):
            x, w, b = rand(t, k), (rand(k, v) if order == 0 else rand(v, k).t()) * k ** -0.5, rand(v)
            labels = torch.randint(v, (t,), device="cuda", generator=g)
            labels[::5] = -100
            if t == 1:
                labels[0] = 3
            check_entropy(x, w, b, labels, str(dtype)[6:], "sum", 1.0, limit)
            clear(("entropy", t, k, v, dtype, limit))
    sizes = [1, 255, 256, 257, 3, 0, 2048, 2049, 7, 8192 * 3 + 5, 40000]
    for bits in (32, 8):
        for offset in (0, 1):
            for many in (1, 12):
                params = [rand(n + offset)[offset:] for n in sizes * many]
                before = [p.clone() for p in params]
                grads = [None if i == 4 else torch.sign(rand(n + offset))[offset:] for i, n in enumerate(sizes * many)]
                opt = ax.AdamW(params, lr=0.25, weight_decay=0.0, state_bits=bits)
                opt.step(grads)
                for p, q, d in zip(params, before, grads):
                    want = q.double() - (0 if d is None else 0.25 * d.double())
                    assert p.numel() == 0 or float((p.double() - want).abs().max()) < 0.03
                opt.step(grads)
                clear(("adamw", dtype, bits, offset))
print("violations 0")
"""


def test_checked_flavour_finds_no_violation(built):
    env = dict(os.environ, AXC_LIBRARY_FLAVOUR="check")
    r = subprocess.run([sys.executable, "-c", CHILD % (ROOT, os.path.join(ROOT, "tests"))], env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    assert "violations 0" in r.stdout
