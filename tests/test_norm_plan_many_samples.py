"""CPU: what the plan of group norm (csrc/axc_norm_plan.h, compiled here) chooses for many samples of few places, where the form that reads its tensors twice
has a block for every sample and group between its two passes: measured, it took 10 to 50 times as long as resident spans."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include "axc_norm_plan.h"
int main()
{
    // samples, places, channels, groups, and whether the tensors are read twice
    const long long shapes[][5] = {{200704, 1, 256, 32, 0}, {50000, 1, 256, 32, 0}, {16384, 16, 64, 8, 0}, {20000, 1, 64, 64, 0}, {6263, 3, 765, 51, 0}, {8192, 9, 96, 3, 0},
                                   {4096, 1, 768, 1, 0}, {1 << 20, 2, 48, 3, 0}, {256, 3136, 256, 32, 0}, {2, 262144, 128, 32, 1}, {1, 20000, 520, 2, 1}, {2, 1100000, 1024, 2, 1}};
    int wrong = 0;
    for (const auto &v : shapes)
        for (int backward = 0; backward < 2; ++backward)
            for (int residual = 0; residual < 2; ++residual) {
                const axc::NormShape s = {v[0], v[1], v[2], v[3], 2, true};
                const axc::NormPlan p = axc::norm_plan(s, (backward ? 2 + residual : 1) * 2, (backward ? 3 + 2 * residual : 2 + residual) * 2, backward, 148);
                if (p.resident == (v[4] != 0)) std::printf("%lld %lld %lld %lld backward %d residual %d: resident %d\n", v[0], v[1], v[2], v[3], backward, residual, int(p.resident)), ++wrong;
            }
    return wrong != 0;
}
"""


def test_many_samples_stay_resident(tmp_path):
    source, program = tmp_path / "plan.cpp", str(tmp_path / "plan")
    source.write_text(PROGRAM)
    subprocess.run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-I" + os.path.join(ROOT, "tf-approximate_b200", "csrc"), str(source), "-o", program], check=True)
    r = subprocess.run([program], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
