"""The bound that the GPU tests hold the paged decode to, against its products
restated on the CPU: three terms are within it, two are not."""
import numpy as np
import pytest

from oracle import oracle as O
from paged_products import restated, terms, tight64
from paged_util import rounded


def test_three_terms_are_the_value():
    x = np.concatenate([O.fill_normal((1000,), 1, "x"), np.float32([0.0, 1.0, -3.0e38, 1e-30, 16777215.0])])
    assert np.array_equal(sum(t.astype(np.float64) for t in terms(x, 3)), x.astype(np.float64))
    assert (sum(t.astype(np.float64) for t in terms(x, 2)) != x).mean() > 0.9


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("n,size", [(1, 1.0), (2, 1.0), (8, 1.0), (17, 1.0), (33, 1.0), (100, 1.0), (300, 1.0), (300, 8.0), (300, 100.0), (1000, 2.0)])
def test_two_terms_exceed_the_bound(dim, n, size):
    heads, kv = 12, 2
    q = (size * O.fill_normal((heads, dim), n, "q")).astype(np.float32)
    k, v = (rounded(O.fill_normal((n, kv, dim), n + dim, name), "bf16").astype(np.float64) for name in "kv")
    want, bound = tight64(q.astype(np.float64), k, v, n - 1)

    def worst(query_terms, weight_terms):
        return (np.abs(restated(q, k, v, query_terms, weight_terms) - want) / bound).max()

    assert worst(3, 3) <= 1.0
    if n >= 33:             # (of one key the weight is 1, of two nearly)
        assert worst(2, 3) > 1.0
    if 8 <= n <= 33:        # (the sum over more positions rounds as much itself)
        assert worst(3, 2) > 1.0
