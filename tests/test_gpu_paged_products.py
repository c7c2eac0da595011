"""GPU accuracy of the paged decode's products: within a bound that the loss of
one of their three terms exceeds (test_paged_products.py), over lengths, dims,
query forms, and head groups that do not fill up evenly."""
import numpy as np
import pytest

from gpu_util import dev_f32, host, say
from oracle import oracle as O
from paged_products import tight64
from paged_util import Cache, rounded
from test_gpu_paged import _dev, _options

pytestmark = pytest.mark.gpu


def _check(gpu, cache, q, dtype, opt, max_length=None, **kw):
    import torch
    out = torch.full((q.shape[0], q.shape[1], cache.dim), 7.0, device="cuda")
    say("paged decode", dict(lengths=cache.lengths[:8], heads=q.shape[1], kv=cache.kv, dim=cache.dim, dtype=dtype), kw)
    gpu.paged_decode(_dev(q, dtype), out, *cache.device(), max_length=max_length,
                     q_norm=None if opt["gamma"] is None else dev_f32(opt["gamma"]),
                     freqs=None if opt["freqs"] is None else dev_f32(opt["freqs"]), interleaved=opt["interleaved"],
                     amplitude=opt["amplitude"], **kw)
    got, worst = host(out), 0.0
    for b, n in enumerate(cache.lengths):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        k, v = cache.rows(b)
        want, bound = tight64(q[b].astype(np.float64), k, v, n - 1, **opt, **kw)
        worst = max(worst, (np.abs(got[b] - want) / bound).max())
    print("worst error of the bound:", worst)
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("size", [1.0, 8.0, 100.0, 3000.0])
def test_products(gpu, dim, size):
    """queries as they are, neither normed nor turned; at the largest, scores of +-60000"""
    cache = Cache([8, 17, 33, 64, 100, 400, 2, 1], 2, 16, dim, dim)
    q = rounded(size * O.fill_normal((8, 12, dim), dim, "q"), "f32")
    _check(gpu, cache, q, "f32", _options(dim, 1, False, 0))


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("norm,rot,interleaved,amplitude", [(True, 1.0, False, 1.0), (True, 1.0, True, 1.25),
                                                            (False, 0.5, False, 1.0), (True, 0.25, True, 0.75)])
def test_products_of_normed_and_turned_queries(gpu, dim, norm, rot, interleaved, amplitude):
    cache = Cache([9, 33, 100, 500], 2, 16, dim, dim + 1)
    opt = _options(dim, 2, norm, int(dim * rot) // 2 * 2, interleaved, amplitude)
    _check(gpu, cache, rounded(O.fill_normal((4, 12, dim), 3, "q"), "f32"), "f32", opt)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(17, 1), (33, 1), (38, 2), (15, 5)])
@pytest.mark.parametrize("lengths", [[33, 100, 0, 7, 90] * 13, [9000], [3000, 2]])
def test_groups_that_do_not_fill_up(gpu, dim, heads, kv, lengths):
    """17 query heads a kv head are two groups of 9 and 8, 33 three of 11, 19 two of 10 and 9; pairs within a wave's
    run, joined by the last workgroup to arrive (many short sequences) and by a second launch (few long ones)"""
    cache = Cache(lengths, kv, 16, dim, heads)
    q = rounded(O.fill_normal((len(lengths), heads, dim), heads, "q"), "f32")
    _check(gpu, cache, q, "f32", _options(dim, 4, False, 0), max_length=max(lengths))


@pytest.mark.parametrize("window", [33, 100])
def test_products_in_a_window(gpu, window):
    cache = Cache([1000, 40, 333], 2, 24, 64, 5)
    q = rounded(O.fill_normal((3, 12, 64), 6, "q"), "f32")
    _check(gpu, cache, q, "f32", _options(64, 7, True, 32, True), window=window)
