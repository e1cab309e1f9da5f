"""The library holds the decode kernels that a call reaches: mode and waves a workgroup as the launches choose them."""
import re

from abridgekv_amd._lib import LIB_PATH


def test_decode_kernels():
    """Template arguments (KV heads a workgroup, waves that share a split, mode): plain 0, window 1, scored 2, whole 3. A plain
    decode of one split takes the forms that longer ones take."""
    names = re.findall(rb"decode_attn_kernelILi(\d+)ELi(\d+)ELi(\d+)E", LIB_PATH.read_bytes())
    assert {tuple(int(x) for x in n) for n in names} == {
        (2, 1, 0), (1, 4, 0), (2, 1, 1), (1, 4, 1), (1, 8, 1), (2, 1, 2), (1, 4, 2), (1, 8, 2), (1, 8, 3)}
