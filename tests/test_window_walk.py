"""The key-tile walk and the dK/dV work plan of the sliding-window kernels (csrc/window_walk.h, built for the host) against
the definition: every visible (query, key) pair falls to exactly one tile, no hidden one to any."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest

from oracle import window as ow

ROOT = Path(__file__).resolve().parent.parent
BIG = (1 << 31) - 1


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    so = tmp_path_factory.mktemp("window_walk") / "harness.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-fsanitize=undefined",
                    "-fno-sanitize-recover=undefined", f"-I{ROOT / 'abridgekv_amd' / 'csrc'}",
                    str(ROOT / "tests" / "window_walk_harness.cpp"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.window_counts.restype = lib.dkv_counts.restype = C.c_long
    return lib


def _sizes():
    yield from [(1, 1, 0), (1, 1, 1), (64, 64, 0), (65, 64, 64), (200, 1, 0), (200, BIG, BIG), (200, BIG, 0),
                (200, 1, BIG), (129, 65, 1), (500, 128, 4), (777, 129, 17), (640, 63, 130), (640, 64, 128), (640, 2, 65)]
    r = random.Random(5)
    for _ in range(60):
        yield (r.randint(1, 700), r.choice([1, 2, 63, 64, 65, 128, r.randint(1, 800)]), r.choice([0, 1, 4, 64, r.randint(0, 800)]))


def test_walk_covers_the_window_once(harness):
    r = random.Random(7)
    for n, window, sinks in _sizes():
        for base in {0, r.randint(0, n - 1)}:
            got = np.zeros((n, n), np.uint8)
            tiles = harness.window_counts(n, base, window, sinks, got.ctypes.data_as(C.c_void_p))
            want = ow.visible(np.arange(n), n, window, sinks)
            assert tiles > 0, (n, base, window, sinks)
            assert (got[base:] == want[base:]).all() and not got[:base].any(), (n, base, window, sinks)
            # bounded by the window: at most the sinks' tiles and two more than the windows of 64 rows fill
            most = -(-min(sinks, n) // 64) + (min(window, n) + 63) // 64 + 2
            assert tiles <= most * -(-(n - base) // 64), (n, base, window, sinks)


def test_dkv_plan_covers_the_window_once(harness):
    r = random.Random(11)
    for S, window, sinks in _sizes():
        for n in {S, 0, r.randint(0, S)}:
            got = np.zeros((max(n, 1), max(n, 1)), np.uint8)
            items = harness.dkv_counts(S, n, r.choice([1, 3]), window, sinks, got.ctypes.data_as(C.c_void_p))
            assert items > 0, (S, n, window, sinks)
            if n:
                assert (got == ow.visible(np.arange(n), n, window, sinks)).all(), (S, n, window, sinks)


def test_workspace_grows_with_the_sinks_not_with_the_rows():
    from abridgekv_amd._lib import lib
    size = lib().abkv_window_bwd_workspace_size
    rows = 2 * 8192 * 32 * 4
    assert size(1, 8192, 512, 0) <= rows + 4096
    assert rows < size(1, 8192, 512, 4) <= rows + (384 + 1) * 8 * 65536 + 4096
    # every key a sink: one far part for each tile at least, at most twice the bound
    assert size(1, 8192, 512, 1 << 30) <= rows + 2 * (384 + 128) * 8 * 65536 + 4096
    assert size(0, 64, 1, 0) == size(1, 0, 1, 0) == size(1, 64, 0, 0) == size(1, 64, 1, -1) == 0
