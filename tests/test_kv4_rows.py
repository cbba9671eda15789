"""Which token a row of a call is (kv4_rows_seq of csrc/kv4_layout.h, compiled
for the host): whatever cu_rows and seq_lens hold, row cu[b] + i is token
len - (cu[b+1] - cu[b]) + i."""
import ctypes
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INT_MAX, INT_MIN = 2 ** 31 - 1, -2 ** 31
MOST_ROWS = 2 ** 31 - 4097


@pytest.fixture(scope="module")
def seq(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("kv4") / "rows_probe.so")
    subprocess.run([gxx, "-O1", "-std=c++17", "-fPIC", "-shared", "-ftrapv", "-I",
                    os.path.join(ROOT, "tensor-bridge_b200", "csrc"),
                    os.path.join(ROOT, "tests", "kv4_rows_probe.cpp"), "-o", out], check=True, timeout=120)
    lib = ctypes.CDLL(out)

    def call(rows, width, shift, cu0, cu1, ln):
        res = (ctypes.c_int * 6)()
        lib.p_rows_seq(rows, width, shift, cu0, cu1, ln, res)
        return tuple(res)

    return call


def test_rows_inside_keep_their_tokens(seq):
    """30 rows of a sequence of 60 tokens, ten of them inside."""
    assert seq(100, 4, 5, 90, 120, 60) == (90, 10, 60, 30, 0, 1)
    assert seq(100, 4, 5, -3, 5, 60) == (0, 5, 60, 55, 0, 1)    # the first three are outside
    assert seq(100, 4, 5, -3, 105, 60) == (0, 100, 60, -45, 0, 1)
    assert seq(100, 4, 5, 90, 100, 60) == (90, 10, 60, 50, 0, 0)
    assert seq(100, 4, 5, 100, 100, 60)[5] == 0
    assert seq(100, 4, 5, 50, 40, 60)[1::4] == (0, 1)           # decreasing: no rows
    assert seq(100, 4, 5, 101, 103, 60)[1::4] == (0, 1)         # all outside


def test_positions_at_the_edges(seq):
    edge = [INT_MIN, INT_MIN + 1, -5000, -7, -1, 0, 1, 5, 63, 64, 65, 1000, INT_MAX - 4096, INT_MAX]
    for rows in (0, 1, 64, MOST_ROWS):
        for cu0 in edge:
            for cu1 in edge:
                for ln in edge:
                    first, n, length, pos0, bad, cut = seq(rows, 4, 4, cu0, cu1, ln)
                    assert 0 <= first <= rows and 0 <= n <= rows - first
                    assert 0 <= length <= 64 and bad == (ln < 0 or ln > 64)
                    assert cut == (cu0 < 0 or cu1 > rows or cu1 < cu0)
                    if n == 0:
                        continue
                    want = max(ln, 0) - (cu1 - cu0) + (first - cu0)
                    assert pos0 == max(want, INT_MIN + 4096)
                    assert pos0 == want or pos0 + n - 1 < 0
