"""One token's attention over bf16 pages with its scores capped or biased, against float64."""
import numpy as np
import pytest

from gpu_util import dev_bf16, dev_f32, host, say
from oracle import oracle as O
from paged_q4_util import scored64
from paged_util import Cache, rounded

pytestmark = pytest.mark.gpu


def dev(x, dtype):
    return dev_bf16(O.pack_bf16(x)) if dtype == "bf16" else dev_f32(x)


def decoded(gpu, cache, q, dtype, slopes=None, **how):
    import torch
    out = torch.full((len(cache.lengths), q.shape[1], cache.dim), 5.0, device="cuda")
    gpu.paged_decode(dev(q, dtype), out, *cache.device(), slopes=None if slopes is None else dev_f32(slopes), **how)
    return host(out)


def check(cache, got, q, **how):
    for b, n in enumerate(cache.lengths):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        want, bound = scored64(q[b], *cache.rows(b), n - 1, **how)
        assert (np.abs(got[b] - want) <= bound).all(), (b, n, (np.abs(got[b] - want) / bound).max())


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cap,biased,window", [(50.0, False, 0), (1.5, False, 0), (0.0, True, 0), (30.0, True, 70)])
def test_scores_capped_and_biased(gpu, dim, dtype, cap, biased, window):
    cache = Cache([1, 0, 31, 32, 33, 700], 2, 12, dim, 51)
    q = rounded(3 * O.fill_normal((6, 6, dim), 8, "q"), dtype)
    slopes = (2.0 ** -np.arange(1, 7)).astype(np.float32) if biased else None
    say("paged_decode scored", dim, dtype, cap, biased, window)
    got = decoded(gpu, cache, q, dtype, slopes, cap=cap, window=window)
    check(cache, got, q, cap=cap, slopes=slopes, window=window)


def test_slopes_of_a_group_and_of_many_groups(gpu):
    """24 heads of one key head are two groups; each head has its own slope"""
    cache = Cache([600, 90], 1, 16, 64, 52, "position")
    q = O.fill_normal((2, 24, 64), 8, "q")
    slopes = np.linspace(0.001, 0.7, 24).astype(np.float32)
    say("paged_decode slopes")
    check(cache, decoded(gpu, cache, q, "f32", slopes), q, slopes=slopes)


def test_negative_and_zero_slopes(gpu):
    cache = Cache([200], 2, 16, 64, 53)
    q = O.fill_normal((1, 2, 64), 8, "q")
    slopes = np.array([-0.05, 0.0], np.float32)
    say("paged_decode negative slopes")
    check(cache, decoded(gpu, cache, q, "f32", slopes), q, slopes=slopes)


def test_a_large_cap_changes_little_and_none_nothing(gpu):
    cache = Cache([300, 40], 2, 16, 128, 54)
    q = O.fill_normal((2, 8, 128), 8, "q")
    say("paged_decode cap limits")
    plain = decoded(gpu, cache, q, "f32")
    check(cache, plain, q)
    check(cache, decoded(gpu, cache, q, "f32", cap=1e4), q, cap=1e4)
    zero = decoded(gpu, cache, q, "f32", np.zeros(8, np.float32))
    check(cache, zero, q)


def test_scores_far_past_the_cap(gpu):
    """a tanh that is 1: the weights of the keys past it are equal"""
    cache = Cache([64], 1, 16, 64, 55)
    q = (1e4 * O.fill_normal((1, 2, 64), 8, "q")).astype(np.float32)
    say("paged_decode saturated")
    got = decoded(gpu, cache, q, "f32", cap=3.0)
    assert np.isfinite(got).all()
    keys, values = cache.rows(0)
    for h in range(2):
        s = 3.0 * np.tanh(keys[:, 0] @ q[0, h].astype(np.float64) / 8 / 3.0)
        w = np.exp(s - s.max())
        # the saturated tanh is exact; none of these scores is near 0
        np.testing.assert_allclose(got[0, h], w / w.sum() @ values[:, 0], atol=64 * 2.0 ** -24 * np.abs(values).max())


def test_captured(gpu):
    import torch
    cache = Cache([500, 20], 2, 16, 128, 56)
    pools = cache.device()
    q, out, slopes = torch.randn((2, 8, 128), device="cuda"), torch.empty((2, 8, 128), device="cuda"), \
        torch.rand(8, device="cuda")
    say("paged_decode scored, captured")
    work = gpu.paged_decode_workspace(q, out, *pools)

    def step():
        gpu.paged_decode(q, out, *pools, workspace=work, cap=20.0, slopes=slopes)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        q.normal_()
        slopes.uniform_()
        graph.replay()
        again = torch.empty_like(out)
        gpu.paged_decode(q, again, *pools, cap=20.0, slopes=slopes)
        torch.cuda.synchronize()
        assert torch.equal(out, again)
