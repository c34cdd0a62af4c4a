"""CPU: the rows of a cut query tile's records (csrc/paged_records.h), enumerated."""
import ctypes as C
import os
import subprocess

import pytest

from tests.conftest import ROOT

SOURCE = r"""
#include "paged_records.h"
#include <cstdio>
#include <cstring>
using namespace mlzc::paged;
// For a piece of n tokens of a call of `tokens`: every row has a place of its own within the
// record, and the place's token and head are the row's.  0, or what is wrong.
extern "C" int check(int tokens, int n, int G, int ns) {
    const int tq = 128 / G, rows = record_rows(tokens, G, tq, ns);
    bool seen[256] = {};
    if (rows > 256) return 1;
    for (int tile = 0; tile < ns; ++tile)
        for (int row = 0; row < tq * G; ++row) {
            const int tok = tile * tq + row / G;
            if (tok >= n) continue;
            const int at = record_row(tile, row, tq, G);
            if (at < 0 || at >= rows) return 2;
            if (seen[at]) return 3;
            seen[at] = true;
            if (at / G != tok || at % G != row % G) return 4;   // as the merge reads it
        }
    return 0;
}
"""


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    d = tmp_path_factory.mktemp("records")
    (d / "records.cpp").write_text(SOURCE)
    so = str(d / "records.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "mlz_b200", "csrc"),
                    str(d / "records.cpp"), "-o", so], check=True)
    f = C.CDLL(so).check
    f.argtypes = [C.c_int] * 4
    return f


@pytest.mark.parametrize("ns", [1, 2])
def test_every_row_has_a_place_in_its_record(check, ns):
    bad = []
    for G in range(1, 129):
        most = (128 // G) * ns
        for tokens in range(1, 262):
            # pieces of one sequence's tokens: full, or the rest behind full ones
            for n in {min(tokens, most), tokens % most or most, 1}:
                if n <= tokens and (why := check(tokens, n, G, ns)):
                    bad.append((G, tokens, n, why))
    assert not bad, f"{len(bad)} of them, the first: {bad[:8]}"
