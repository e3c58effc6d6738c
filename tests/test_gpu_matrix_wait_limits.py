"""GPU: what the matrix kernels do when their waits run out.  The debug flavour lets a test set the limit to nothing: every kernel must
finish, the status word must say 3, a checked call must raise, and with the limit back the same calls must give the same bits as before."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r"""
import ctypes as C, sys
import torch
sys.path.insert(0, %r)
import tf_approximate_b200 as ax
from tf_approximate_b200 import _lib
L = _lib.load()
rec = (C.c_uint32 * 4)()
assert L.axc_debug_bounds_record(0, rec) == 0, "not the debug flavour"
g = torch.Generator(device="cuda").manual_seed(0)
rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
calls = []
# pairs of CTAs, lone CTAs with wide and narrow tiles, split sums, sums that are taken out on the way
for dtype in (torch.float32, torch.bfloat16, torch.float16):
    for t, k, n, act in ((2100, 136, 4500, None), (300, 4096, 200, "silu"), (64, 64, 20, "relu"), (600, 200, 1000, "relu")):
        x, w, dy = rand(t, k).to(dtype), rand(k, n).to(dtype), rand(t, n).to(dtype)
        _, kept = ax.dense_forward(x, w, None, None, act)
        calls.append(lambda x=x, w=w, act=act: ax.dense_forward(x, w, None, None, act, check=True)[:1])
        calls.append(lambda x=x, w=w, act=act, dy=dy, kept=kept: ax.dense_backward(dy, x, w, kept, act, check=True)[:2])
    # few logits, kept exponentials, pieces of the classes
    for t, v, limit in ((100, 300, None), (1600, 900, None), (300, 900, 1)):
        x, w, b, labels = rand(t, 64).to(dtype), rand(64, v).to(dtype), rand(v), torch.randint(v, (t,), device="cuda", generator=g)
        calls.append(lambda x=x, w=w, b=b, labels=labels, limit=limit: ax.dense_cross_entropy_gradients(x, w, labels, b, scratch_limit=limit, check=True))
want = [call() for call in calls]
for i, call in enumerate(calls):
    assert L.axc_debug_matrix_wait_polls(0, 0) == 0
    try:
        call()
        raise SystemExit("call %%d: a wait that ran out was not reported" %% i)
    except ax.InternalError as e:
        assert "status 3" in str(e), str(e)
    torch.cuda.synchronize()
    assert L.axc_debug_matrix_wait_polls(0, -1) == 0
    assert all(torch.equal(a, b) for a, b in zip(call(), want[i])), i
assert L.axc_debug_bounds_record(0, rec) == 0
print("violations", rec[0], "site", rec[1], "value", rec[2] | (rec[3] << 32))
assert rec[0] == 0
"""


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_reported(built):
    env = dict(os.environ, AXC_LIBRARY_FLAVOUR="check")
    r = subprocess.run([sys.executable, "-c", CHILD % ROOT], env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    assert "violations 0" in r.stdout


def test_normal_build_has_no_wait_limit_to_set(built):
    from tf_approximate_b200 import _lib
    assert _lib.load().axc_debug_matrix_wait_polls(0, 0) == 12       # Unimplemented
