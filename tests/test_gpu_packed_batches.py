"""Packed attention over batches as serving has them: histories of unlike lengths, places without tokens, windows that
leave little of a long history, grids that do not go evenly round the eight XCDs."""
import numpy as np
import pytest

from gpu_util import host, say
from oracle import oracle as O
from packed_util import document64
from paged_util import rounded
from test_gpu_packed import dev, run, vector

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
def test_one_long_history_among_short_ones(gpu, dtype, out):
    """split and not, by what the documents' keys are on average"""
    run(gpu, [5, 9, 3, 1, 7], 8, 2, 128, dtype, out, past=[40, 9000, 300, 0, 17])
    run(gpu, [3] * 30 + [11], 8, 2, 64, dtype, out, past=[20] * 30 + [6000])


@pytest.mark.parametrize("places", [6, 60])
def test_a_batch_padded_with_places_of_no_tokens(gpu, places):
    """with places enough, as many workgroups as a split would make: not split, and the same results"""
    run(gpu, [16, 3, 0, 8] + [0] * places, 32, 8, 128, "bf16", "f32", past=[3000, 2000, 0, 1500] + [0] * places)


@pytest.mark.parametrize("window", [1, 64, 600, 2500])
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
def test_chunks_whose_window_leaves_little(gpu, window, dtype, out):
    run(gpu, [32], 32, 8, 128, dtype, out, past=[9000], window=window, workspace=True)
    run(gpu, [32, 5], 8, 2, 256, dtype, out, past=[5000, 2000], window=window, prefix=[4500, 2005])


@pytest.mark.parametrize("heads,kv,new", [(4, 1, [33] * 3), (12, 12, [40]), (5, 5, [129, 130, 1]), (3, 3, [700])])
def test_grids_that_are_no_multiple_of_eight(gpu, heads, kv, new):
    """(slots times kv heads): 6, 12, 25 and 18 workgroups"""
    slots = sum(new) * (heads // kv) // 128 + len(new)
    assert slots * kv % 8
    run(gpu, new, heads, kv, 128, "bf16", "bf16")


def test_a_captured_window_takes_the_workspace_of_none(gpu):
    """the query without a window is enough for calls with one"""
    import torch
    n, past, H, KV, D = 8, 4000, 8, 2, 128
    q, k, v = (rounded(O.fill_normal((m, h, D), 7, s), "bf16") for m, h, s in ((n, H, "q"), (n + past, KV, "k"), (n + past, KV, "v")))
    tensors = dev(q, "bf16"), dev(k, "bf16"), dev(v, "bf16"), torch.zeros((n, H, D), device="cuda")
    how = dict(starts=vector([0, n]), key_starts=vector([0, n + past]))
    say("packed captured window")
    work = gpu.packed_attention_workspace(*tensors, **how)
    assert work.numel()
    for window in (0, 2000, 100):
        gpu.packed_attention(*tensors, **how, window=window, workspace=work)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gpu.packed_attention(*tensors, **how, window=window, workspace=work)
        want, bound = document64(q, k, v, "bf16", "f32", window=window)
        for _ in range(3):
            tensors[3].fill_(5.0)
            graph.replay()
            torch.cuda.synchronize()
            assert (np.abs(host(tensors[3]) - want) <= bound).all()
