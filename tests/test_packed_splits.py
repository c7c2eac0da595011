"""How far a packed attention splits its keys, told by its workspace, without a GPU."""
import ctypes as C

import pytest

import aigpu

PTR = 1 << 40


def splits(count, keys, documents=1, heads=32, kv=8, dim=128, window=0):
    args = aigpu.AiGpuPackedAttention(q=PTR, k=2 * PTR, v=3 * PTR, out=4 * PTR, starts=PTR, keyStarts=PTR, inType=1,
                                      outType=1, count=count, keyCount=keys, documents=documents, heads=heads,
                                      kvHeads=kv, dim=dim, window=window)
    need = aigpu.lib().aigpu_packed_attention_workspace(C.byref(args))
    record = 128 * (dim + 2) * 4 * kv * (count * (heads // kv) // 128 + documents)
    assert need % record == 0
    return need // record or 1


def test_keys_are_split_from_512_on():
    assert splits(32, 511) == 1 and splits(32, 1023) == 1 and splits(32, 1024) == 2
    assert splits(32, 30032) == 58 and splits(4, 30032 * 4, documents=4) == 16


@pytest.mark.parametrize("window,most", [(1, 1), (64, 1), (512, 1), (1000, 2), (4096, 8), (20000, 39), (40000, 58)])
def test_a_window_leaves_fewer_keys_to_split(window, most):
    """32 tokens behind 30000 keys see window + 32 of them: a split has 512 of those at the least, and a workspace
    for calls without a window holds the records of any"""
    assert splits(32, 30032, window=window) == most <= splits(32, 30032)
