"""CPU: how group norm's kernels cut up their tensors, and every thread's way through its part, for random shapes: nothing left out, nothing twice,
nothing outside, within the shared memory that the launch asks for (csrc/axc_norm_plan.h, compiled here)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_value_once(tmp_path):
    program = str(tmp_path / "norm_plan_check")
    subprocess.run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-I" + os.path.join(ROOT, "tf-approximate_b200", "csrc"),
                    os.path.join(ROOT, "tests", "norm_plan_check.cpp"), "-o", program], check=True)
    r = subprocess.run([program, "500"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
