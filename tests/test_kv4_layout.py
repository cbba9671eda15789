"""Where the cache's kernels may go (csrc/kv4_layout.h, compiled for the host):
rows and lengths that a call's device arrays hold, pages, and the chunks of
tokens that a block of rows visits."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INT_MAX, INT_MIN = 2 ** 31 - 1, -2 ** 31


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("kv4") / "probe.so")
    subprocess.run([gxx, "-O1", "-std=c++17", "-fPIC", "-shared", "-ftrapv", "-I",
                    os.path.join(ROOT, "tensor-bridge_b200", "csrc"),
                    os.path.join(ROOT, "tests", "kv4_layout_probe.cpp"), "-o", out], check=True, timeout=120)
    lib = ctypes.CDLL(out)
    lib.p_offset.restype = ctypes.c_ulonglong
    lib.p_offset.argtypes = [ctypes.c_ulonglong] + [ctypes.c_int] * 4
    return lib


def seq(probe, rows, width, shift, cu0, cu1, ln):
    out = (ctypes.c_int * 5)()
    probe.p_seq(rows, width, shift, cu0, cu1, ln, out)
    return tuple(out)


def test_rows_and_lengths_stay_inside(probe):
    edge = [INT_MIN, -7, -1, 0, 1, 5, 63, 64, 65, 1000, INT_MAX]
    for rows in (0, 1, 64):
        for cu0 in edge:
            for cu1 in edge:
                for ln in edge:
                    first, n, length, pos0, bad = seq(probe, rows, 4, 4, cu0, cu1, ln)
                    assert 0 <= first <= rows and 0 <= n <= rows - first
                    assert 0 <= length <= 64
                    assert bad == (ln < 0 or ln > 64)
                    if not bad:
                        assert length == ln and pos0 == ln - n
    assert seq(probe, 100, 8, 5, 10, 13, 200) == (10, 3, 200, 197, 0)


def test_pages_outside_are_refused(probe):
    assert [probe.p_page_ok(5, p) for p in (INT_MIN, -1, 0, 4, 5, INT_MAX)] == [0, 0, 1, 1, 0, 0]
    assert [probe.p_slot_ok(3, p) for p in (-1, 0, 2, 3, INT_MAX)] == [0, 1, 1, 0, 0]
    assert probe.p_page_ok(0, 0) == 0 and probe.p_slot_ok(0, 0) == 0


def test_offsets_pass_32_bits(probe):
    # 2^20 pages of 64 tokens, 8 heads of 128: 73,728 bytes a page
    assert probe.p_offset(73728, 6, 128, (1 << 20) - 1, 7) == ((1 << 20) - 1) * 73728 + 7 * 64 * 144


@pytest.mark.parametrize("shift", [4, 5, 7])
def test_span_covers_what_rows_see_and_little_more(probe, shift):
    rng = np.random.default_rng(shift)
    size = 1 << shift
    buf = (ctypes.c_int * 4096)()
    for _ in range(1500):
        n = int(rng.integers(1, 40))
        length = int(rng.integers(0, 900))
        window = int(rng.choice([0, 0, 1, 5, 31, 32, 33, 200, INT_MAX]))
        sinks = int(rng.choice([0, 1, 4, 32, 33, 100, 2000, INT_MAX]))
        pos0 = length - n
        got = probe.p_span(pos0, length - 1, length, window, sinks, shift, 4096, buf)
        chunks = list(buf[:got])
        assert got >= 1 and chunks == sorted(set(chunks)) and chunks[0] >= 0
        seen = {t >> shift for p in range(pos0, length) for t in range(0, p + 1)
                if window <= 0 or p - t < window or t < sinks}
        assert seen <= set(chunks)
        if seen:  # nothing past the sequence, and only chunks that hold a sink or a row's window
            assert set(chunks) <= {t >> shift for t in range(length)
                                   if window <= 0 or max(pos0, 0) - t < window or t < sinks}
            assert chunks[-1] * size < length
        else:
            assert got == 1


def test_sees(probe):
    for window in (0, 1, 3, INT_MAX):
        for sinks in (0, 2, INT_MAX):
            for pos in range(-2, 9):
                for tok in range(9):
                    want = tok <= pos and (window == 0 or tok > pos - window or tok < sinks)
                    assert bool(probe.p_sees(pos, tok, window, sinks)) == want
