"""The dK/dV work plan of the sliding-window backward with many sinks: the workspace stays bounded, and every pair of key and query
tiles that see one another falls to one item."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from abridgekv_amd._lib import lib
from oracle import window as ow

ROOT = Path(__file__).resolve().parent.parent
SLOTS = 384                                                  # far parts of a launch, and sink tiles that have some


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    so = tmp_path_factory.mktemp("window_plan") / "harness.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-fsanitize=undefined",
                    "-fno-sanitize-recover=undefined", f"-I{ROOT / 'abridgekv_amd' / 'csrc'}",
                    str(ROOT / "tests" / "window_plan_harness.cpp"), "-o", str(so)], check=True)
    return C.CDLL(str(so))


# rows, batch, window, sinks
LAUNCHES = [(8192, 8, 64, 4096), (32768, 4, 64, 16384), (8192, 1, 512, 4), (8192, 3, 512, 8192), (8192, 4, 64, 8191), (777, 3, 129, 17),
            (192, 192, 1, 128), (192, 193, 1, 128), (640, 40, 65, 640), (4096, 6, 300, 64 * 64), (4096, 7, 300, 55 * 64),
            (1 << 20, 60, 1000, 1 << 20), (2000, 2, 2000, 2000)]


@pytest.mark.parametrize("S,B,window,sinks", LAUNCHES)
def test_the_slots_are_bounded(harness, S, B, window, sinks):
    out = (C.c_int * 4)()
    harness.plan(S, B, window, sinks, out)
    items, sink_tiles, parts, slots = out
    assert sink_tiles * B <= SLOTS and sink_tiles * parts * B <= SLOTS
    assert slots * B <= 2 * SLOTS
    rows = 2 * B * 32 * (-(-S // 64) * 64) * 4
    assert rows <= lib().abkv_window_bwd_workspace_size(B, S, window, sinks) <= rows + 2 * SLOTS * 8 * 65536 + 8 * 4 * SLOTS + 512


@pytest.mark.parametrize("S,B,window,sinks", [x for x in LAUNCHES if x[0] <= 8192])
def test_every_pair_falls_to_one_item(harness, S, B, window, sinks):
    tiles = -(-S // 64)
    for n in {S, S // 3, 65, 1, 0}:
        got = np.zeros((tiles, tiles), np.uint8)
        harness.tile_counts(S, n, B, window, sinks, got.ctypes.data_as(C.c_void_p))
        k, q = np.arange(tiles)[:, None], np.arange(tiles)[None]
        last = np.minimum(64 * q + 63, n - 1)                # a tile of rows sees one of keys from its first key on
        see = (64 * q < n) & (64 * k <= last) & ((64 * q - (64 * k + 63) < window) | (64 * k < sinks))
        assert (got == see).all(), n


@pytest.mark.gpu
@pytest.mark.parametrize("S,window,sinks", [(192, 1, 128), (200, 70, 190)])
def test_gradients_without_parts(S, window, sinks):
    """More sink tiles than slots: against the oracle, and against the same sequences in a batch that has parts."""
    from abridgekv_amd import ops
    gen = torch.Generator().manual_seed(S)
    few, B = 3, 200
    part = [torch.randn((few, S, h, 128), generator=gen).to(torch.bfloat16) for h in (32, 8, 8, 32)]
    lens = [S, 130, 65]
    q, k, v, g = (t.cuda().repeat(-(-B // few), 1, 1, 1)[:B] for t in part)
    sl = torch.tensor((lens * B)[:B], dtype=torch.int32, device="cuda")
    lse = torch.empty((B, 32, S), device="cuda")
    low = torch.empty((B, S, 32, 128), dtype=torch.float8_e5m2, device="cuda")
    out, _ = ops.window_attention(q, k, v, window, sinks, seq_lens=sl, lse=lse, out_low=low)
    got = ops.window_attention_backward(q, k, v, out, lse, g, window, sinks, seq_lens=sl, out_low=low)
    for b, n in enumerate(lens):
        for t in part:
            t[b, n:] = 0
    want = ow.window_backward(*(t.double().numpy() for t in part), lens, window, sinks, 128 ** -0.5, bounds=True)
    for name, x, d, tol in zip(("dq", "dk", "dv"), got, want[::2], want[1::2]):
        for b in (0, 1, 2, B - 2, B - 1):
            assert (np.abs(x[b].double().cpu().numpy() - d[b % few]) <= tol[b % few]).all(), (name, b)
        assert torch.equal(x[:few], x[few: 2 * few]), name
