"""GPU: group norm, dropout and the 8-bit dense layer in the debug flavour (libaxconv_check.so), in which every global index and every computed
shared-memory address is checked before use, over sizes and layouts that reach every kernel, against the bounds of the operators' own tests; and the
8-bit layer's waits, when they run out."""
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
import test_gpu_dense_8bit as t8, test_gpu_dropout as td, test_gpu_group_norm as tn

def clear(what):
    assert L.axc_debug_bounds_record(0, rec) == 0
    assert rec[0] == 0, (what, rec[0], "site", rec[1], "value", rec[2] | (rec[3] << 32))

for dtype in ("float32", "bfloat16", "float16"):
    for i, (shape, groups) in enumerate(tn.SHAPES + tn.LARGE[:3]):
        x, scale, offset, residual, grad = tn.make(shape, dtype, "float32" if i %% 2 else dtype)
        tn.check_norm(x, groups, scale if i %% 5 else None, offset, residual if i %% 3 else None, (None, "silu", "gelu", "relu")[i %% 4], grad, k=64 if i < len(tn.SHAPES) else 1024)
        clear(("group norm", shape, groups, dtype))
    tn.test_strides_and_alignment(True, dtype) if dtype != "float16" else None
    clear(("group norm, strides", dtype))
    for shape in ((1,), (9,), (256, 2048), (1001, 777)):
        x, r = [torch.randn(shape, device="cuda").to(getattr(torch, dtype)) for _ in range(2)]
        td.check_dropout(x, 0.3, 5, 6)
        td.check_dropout(x, 0.3, 5, 6, r)
        td.check_dropout(x[1:], 0.3, 5, 6) if x.dim() == 1 and x.numel() > 1 else None
        clear(("dropout", shape, dtype))
    for r, k, u in t8.SIZES + [(2100, 136, 4500), (300, 16400, 200)]:
        x, w, b, res, _ = t8.make(r, k, u, dtype)
        t8.check_dense8(x, *ax.quantize_blocks(w, 128), b, res if r %% 2 else None, "silu")
        clear(("dense_8bit", r, k, u, dtype))
    t8.test_codes_and_scales(True, 129, 127, dtype)
    clear(("codes", dtype))
t8.test_strides_and_alignment(True)
clear("dense_8bit, strides")

# waits that run out: pairs of CTAs, lone CTAs with wide and narrow tiles, split sums
for r, k, u in ((2100, 136, 4500), (300, 4096, 200), (64, 64, 20), (600, 200, 1000)):
    x, w, b, res, _ = t8.make(r, k, u, "bfloat16")
    operands = ax.quantize_blocks(w, 128)
    want = ax.dense_8bit(x, *operands, b, check=True)
    assert L.axc_debug_matrix_wait_polls(0, 0) == 0
    try:
        ax.dense_8bit(x, *operands, b, check=True)
        raise SystemExit("a wait that ran out was not reported")
    except ax.InternalError as e:
        assert "status 3" in str(e), str(e)
    torch.cuda.synchronize()
    assert L.axc_debug_matrix_wait_polls(0, -1) == 0
    assert torch.equal(ax.dense_8bit(x, *operands, b, check=True), want)
clear("waits")
print("violations 0")
"""


def test_checked_flavour_finds_no_violation(built):
    env = dict(os.environ, AXC_LIBRARY_FLAVOUR="check")
    r = subprocess.run([sys.executable, "-c", CHILD % (ROOT, os.path.join(ROOT, "tests"))], env=env, capture_output=True, text=True, timeout=1500)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    assert "violations 0" in r.stdout
