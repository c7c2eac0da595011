"""Rows with infinities and NaN through the norm of an append into 4-bit pages."""
import numpy as np
import pytest

from gpu_util import dev_f32, say
from oracle import oracle as O
from paged_q4_util import CacheQ4
from paged_util import normed, turn
from test_gpu_paged_q4 import appended, check_pool, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rot", [0, 64])
def test_an_infinity_under_the_norm_is_its_own_blocks(gpu, dim, dtype, rot):
    """1 / sqrt(infinity) is 0: the row's finite elements become 0, the infinite one NaN, and with it its block, and
    that of its partner in the rotation; NaN makes NaN of the row; rows beside are as they are"""
    cache = CacheQ4([9], 2, 4, dim, 41, fill=False)
    k, v = rows_of(cache, [9], dtype, 42)
    k[1, 0, 5], k[2, 1, dim - 1], k[4, 0, 40] = np.inf, -np.inf, np.nan
    v[3, 0, 33] = np.inf
    gamma = O.fill_uniform((dim,), 9, "g", 0.5, 1.5)
    freqs = (1e4 ** -(np.arange(rot // 2) / (rot // 2))).astype(np.float32) if rot else None
    say("append_q4 infinities", dim, dtype, rot)
    how = dict(freqs=dev_f32(freqs)) if rot else {}
    before, after, _ = appended(gpu, cache, [9], k, v, dtype, k_norm=dev_f32(gamma), **how)
    with np.errstate(invalid="ignore"):
        exact = turn(normed(k, gamma, float(np.float32(1e-6))), np.arange(9), freqs)
    check_pool(cache, [9], exact, v, before, after, off_border=1e-9)
