"""CPU: the partial sums of the bias's gradient fit into their part of the cross entropy's workspace, for every piece of the classes that a
call walks over; the sizes come from the header that the library itself is built from."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SWEEP = r"""
#include <stdio.h>
#include "axc_pieces.h"
using namespace axc;

// every piece that the walk over the classes has, against the room that the workspace has for one
static long check(long long rows, long long classes, long long piece)
{
    const size_t room = slope_scratch_of_pieces(rows, classes, piece);
    long bad = 0;
    for (long long c0 = 0; c0 < classes; c0 += piece) {
        const long long n = classes - c0 < piece ? classes - c0 : piece;
        const PieceSizes s = piece_sizes(classes, piece);
        if (n != s.n[0] && n != s.n[1]) ++bad;
        if (slope_scratch(rows, n) > room) ++bad;
    }
    return bad;
}

int main()
{
    long bad = 0, sizes = 0, rounded = 0;
    unsigned long long state = 1;
    const long long named[][2] = {{8192, 4850}, {4096, 5119}, {8192, 25087}, {65536, 50257}, {65536, 50265}, {65536, 100277}, {65536, 151936}, {65536, 250002}, {16384, 50257}};
    for (int i = 0; i < 400000; ++i) {
        long long rows, classes;
        if (i < 9) rows = named[i][0], classes = named[i][1];
        else {
            state = state * 6364136223846793005ull + 1442695040888963407ull;
            rows = 1 + (long long)(state >> 33) % (1ll << (1 + (state >> 20) % 18));
            state = state * 6364136223846793005ull + 1442695040888963407ull;
            classes = 1 + (long long)(state >> 33) % (1ll << (1 + (state >> 20) % 19));
        }
        const long long whole = (classes + 63) / 64 * 64;
        bad += check(rows, classes, classes);
        rounded += slope_scratch(rows, classes) > slope_scratch(rows, whole);       // what room for whole segments would not hold
        for (int planes = 1; planes <= 3; planes += 2)
            for (size_t limit = 1; limit <= 4ull << 30; limit = limit * 37 + 1) bad += check(rows, classes, classes_of_piece(rows, whole, planes, limit));
        bad += check(rows, classes, classes_of_piece(rows, whole, 1, 4ull << 30));
        ++sizes;
    }
    printf("%ld %ld %ld\n", sizes, bad, rounded);
    return 0;
}
"""


def test_column_sums_fit_for_every_piece(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("needs g++")
    source, program = tmp_path / "sweep.cpp", tmp_path / "sweep"
    source.write_text(SWEEP)
    subprocess.run([gxx, "-O2", "-std=c++17", "-I" + os.path.join(ROOT, "tf-approximate_b200", "csrc"), str(source), "-o", str(program)], check=True)
    sizes, bad, rounded = map(int, subprocess.run([str(program)], check=True, capture_output=True, text=True, timeout=300).stdout.split())
    assert sizes == 400000 and bad == 0
    assert rounded > 0               # the sizes where the room for the next multiple of 64 is too small are among them
