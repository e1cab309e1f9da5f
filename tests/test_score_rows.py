"""The prompt scores' query rows over the strides that the entry accepts: offsets past 2^31, built for the host with checks of
undefined arithmetic, and the strides that are refused."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

from abridgekv_amd._lib import lib

ROOT = Path(__file__).resolve().parent.parent
TOP_TOKEN, TOP_HEAD = (1 << 24) - 8, (1 << 28) - 8           # the largest strides of 16-byte aligned rows


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    so = tmp_path_factory.mktemp("score_rows") / "harness.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-fsanitize=undefined",
                    "-fno-sanitize-recover=undefined", f"-I{ROOT / 'abridgekv_amd' / 'csrc'}",
                    str(ROOT / "tests" / "score_rows_harness.cpp"), "-o", str(so)], check=True)
    so = C.CDLL(str(so))
    so.piece.restype = C.c_uint
    so.piece.argtypes = [C.c_int, C.c_int, C.c_long, C.c_long, C.c_int]
    so.head_stride_ok.argtypes = [C.c_long]
    return so


@pytest.mark.parametrize("token,head", [(4096, 128), (128, 128 * 777), (TOP_TOKEN, 128), (4096, TOP_HEAD), (TOP_TOKEN, TOP_HEAD),
                                        (0, 0)])
def test_offsets(harness, token, head):
    for row in range(128):
        for limit in (0, 7, 31):
            for p in (0, 15):
                want = 2 * (min(row % 32, limit) * token + row // 32 * head + 8 * p)
                assert harness.piece(row, limit, token, head, p) == want < 1 << 32, (row, limit, p)


def test_head_strides():
    """Below 0 and from 2^28 on refused by the C entry, which has no other use for the sign."""
    one, bad = 1 << 12, 1

    def scores(stride):
        starts, past = (C.c_int32 * 2)(0, 5), (C.c_int32 * 1)(0)
        return lib().abkv_paged_prefill_scores(one, 4096, stride, one, 4, one, 4, 4, C.addressof(starts), C.addressof(past), 1,
                                               64, one, one, 64, 64, 1.0, 0)

    for stride in (-8, -128, -(1 << 28), 1 << 28, 1 << 40, -(1 << 40)):
        assert scores(stride) == bad, stride


@pytest.mark.gpu
def test_rows_far_apart():
    """Queries at the largest strides give the bits of dense ones."""
    from abridgekv_amd import ops
    T, past = 75, 40
    gen = torch.Generator().manual_seed(1)
    q = torch.randn((T, 32, 128), generator=gen).to(torch.bfloat16).cuda()
    cache = torch.randn((8, 2, 16, 8, 128), generator=gen).to(torch.bfloat16).cuda()
    table = torch.arange(8, dtype=torch.int32)[None].cuda()
    # (a head stride of TOP_HEAD is 16 token strides and 120 elements: token t + 16 of head h and token t of head h + 1 would
    # share memory)
    head = 16 * TOP_TOKEN - 1024
    store = torch.empty((T - 1) * TOP_TOKEN + 31 * head + 128, dtype=torch.bfloat16, device="cuda")
    far = store.as_strided((T, 32, 128), (TOP_TOKEN, head, 1))
    far.copy_(q)
    assert torch.equal(far, q)
    got = []
    for rows in (q, far):
        lse = torch.empty((T, 32), device="cuda")
        out, _ = ops.paged_prefill_attention_window(rows, cache, table, [0, T], [past], 1000, lse=lse)
        scores = torch.zeros((1, 8, 128), device="cuda")
        ops.paged_prefill_scores(rows, cache, table, [0, T], [past], lse, scores)
        got.append((out, lse, scores))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    # a query row and head weigh 1 in all, each weight good to about 4e-5
    assert abs(float(got[0][2].double().sum()) - 32 * T) <= 4e-5 * 32 * T * 2
