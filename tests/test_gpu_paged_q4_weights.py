"""One token over 4-bit pages where most of the weights are far below the largest, and queries as large as fp32 has."""
import numpy as np
import pytest

from gpu_util import dev_f32, host, say
from oracle import oracle as O
from paged_q4_util import CacheQ4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch,n,kv", [(1, 131072, 1), (6, 30000, 1), (40, 700, 2), (256, 131072, 8)])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
def test_many_small_weights_beside_a_large_one(gpu, dim, batch, n, kv, place):
    """one key and n - 1 whose scores are 21.6 under its (4e-10 of its weight): the result keeps what they add up to,
    also where one wave takes all of a sequence's positions (the last batch), whose maximum is the one key's then

    The bound: a weight's two fp16 terms leave 2^-40 of the largest weight; a score of 21.6 log2(e) carries the query's
    two terms, a product, the exponential's argument and its result, of 2^-22 and 2^-24. Parts are added to a sum one
    after the other, each rounding by 2^-24 of it: four of each slab of 64 that a wave takes, then at most 768
    workgroups' records of a head in four shares of 192, four shares and four waves, which is 200 for the values and
    200 for the weights. (Records of equal small parts round the same way: no random walk.) And what the wave of the
    largest weight adds to it is below a half step of fp32 in each slab, so that the sum may keep none of it; values
    that are 0 for the one key do without that sum."""
    import torch
    below = 21.6
    at = dict(first=0, middle=n // 2, last=n - 1)[place]
    keys, values = (torch.zeros((n, kv, dim), device="cuda") for _ in "kv")
    keys[at, :, 0] = 7.0                              # values that codes hold: scale 1, code 7
    values[:] = 7.0
    values[at, :, :dim // 2] = 0.0
    pages = -(-n // 64)
    pools = [torch.zeros((pages, kv, 64, w), device="cuda", dtype=t) for _ in "kv"
             for w, t in ((dim // 2, torch.uint8), (dim // 32, torch.float16))]
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    gpu.paged_append_q4(keys, values, *pools, table, torch.tensor([n], dtype=torch.int32, device="cuda"),
                        starts=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    q, out = torch.zeros((batch, 2 * kv, dim), device="cuda"), torch.empty((batch, 2 * kv, dim), device="cuda")
    q[:, :, 0] = below / 7.0
    say("decode_q4 small weights", dim, batch, n, kv, place)
    gpu.paged_decode_q4(q, out, *pools, table.expand(batch, -1).contiguous(),
                        torch.full((batch,), n, dtype=torch.int32, device="cuda"), scale=1.0)
    w = np.exp(-7.0 * float(np.float32(below / 7.0)))
    tail = (n - 1) * w / (1 + (n - 1) * w)
    slabs = -(-batch * kv * (-(-n // 64) + 1) // 1024)     # a wave's, where they are fewest
    score = below * np.log2(np.e) * (2 * 2.0 ** -22 + 4 * 2.0 ** -24) + 8 * 2.0 ** -24
    alike, adds = min(n, 64 * slabs) * w, (400 + 4 * slabs) * 2.0 ** -24
    far = host(out)
    assert (np.abs(far[..., :dim // 2] - 7.0 * tail) <= 7.0 * (n * 2.0 ** -40 + tail * (score + alike + adds))).all()
    assert (np.abs(far[..., dim // 2:] - 7.0) <= 7.0 * (n * 2.0 ** -40 + alike + adds)).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("size", [1e34, 1e35, 1e36, 1e37])
def test_queries_of_any_size(gpu, dim, size):
    """queries near fp32's largest, over keys that keep the scores within it, pick one key; beside such a head, others
    are as they are by themselves"""
    cache = CacheQ4([130, 20], 2, 16, dim, 34, size=1e-3)
    q = O.fill_normal((2, 4, dim), 8, "q")
    large = q.copy()
    large[:, 1::2] *= np.float32(size)
    import torch
    alone, got = (torch.empty((2, 4, dim), device="cuda") for _ in "ab")
    say("decode_q4 large queries", dim, size)
    gpu.paged_decode_q4(dev_f32(q), alone, *cache.device(), scale=1.0)
    gpu.paged_decode_q4(dev_f32(large), got, *cache.device(), scale=1.0)
    np.testing.assert_array_equal(host(got)[:, ::2], host(alone)[:, ::2])
    for b in range(2):
        keys, values = cache.rows(b)
        for h in (1, 3):
            best = (keys[:, h // 2] @ large[b, h].astype(np.float64)).argmax()
            np.testing.assert_allclose(host(got)[b, h], values[best, h // 2], rtol=1e-6, atol=0)
