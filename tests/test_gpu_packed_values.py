"""Values that are not finite, among the documents of a packed attention: as the weighted sum has it, each reaches its
own channel of the tokens that see its row, whichever tiles and splits the rows fall into."""
import numpy as np
import pytest

from gpu_util import host, say
from oracle import oracle as O
from paged_util import rounded
from test_gpu_packed import dev, vector

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("new,past,how", [
    (300, 0, {}), (300, 0, dict(window=45)), (150, 0, dict(prefix=150, window=20)), (21, 1500, dict(window=700)),
])
def test_a_value_that_is_not_finite_reaches_its_channel(gpu, dim, dtype, out, new, past, how):
    """rows in tiles that all of a workgroup's tokens see whole and rows in tiles that a mask cuts; every other channel
    and token keeps the bits that finite values give"""
    import torch
    n, H, KV = new + past, 4, 2
    q, k, v = (dev(rounded(O.fill_normal((m, h, dim), 31, s), dtype), dtype)
               for m, h, s in ((new, H, "q"), (n, KV, "k"), (n, KV, "v")))
    window, prefix = how.get("window", 0), how.get("prefix", 0)
    args = dict(starts=vector([0, new]), key_starts=vector([0, n]), window=window)
    if prefix:
        args["prefix"] = vector([prefix])
    plain, got = (torch.zeros((new, H, dim), device="cuda", dtype=torch.bfloat16 if out == "bf16" else torch.float32)
                  for _ in "ab")
    say("packed wild channels", dim, dtype, out, new, past, how)
    gpu.packed_attention(q, k, v, plain, **args)
    i, j = np.arange(past, n)[:, None], np.arange(n)[None]
    sees = ((j <= i) | (j < prefix)) & ((window == 0) | (i - j < window))
    wild = np.zeros((n, dim), bool)
    vv = v.clone()
    # the first rows and the last, two channels of one row, both infinities and NaN in one channel
    for at, d, bad in ((0, 0, np.nan), (3, dim - 1, np.inf), (n // 2, 5, np.nan), (n // 2, 38, -np.inf),
                       (n - 18, 38, np.inf), (n - 2, dim // 2 + 1, np.nan), (n - 1, 5, np.inf)):
        vv[at, 1, d], wild[at, d] = bad, True
    gpu.packed_attention(q, k, vv, got, **args)
    a, b = host(plain), host(got)
    np.testing.assert_array_equal(a[:, :2], b[:, :2])
    reached = np.broadcast_to((sees[:, :, None] & wild).any(1)[:, None], (new, 2, dim))
    np.testing.assert_array_equal(~np.isfinite(b[:, 2:]), reached)
    np.testing.assert_array_equal(a[:, 2:][~reached], b[:, 2:][~reached])


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
def test_an_infinity_keeps_its_sign(gpu, dtype, out):
    """in tiles that a mask cuts, the first of a document among them"""
    import torch
    n, dim = 20, 128
    q, k, v = (dev(rounded(O.fill_normal((n, 1, dim), 32, s), dtype), dtype) for s in "qkv")
    v[0, 0, 9], v[7, 0, 70], v[11, 0, 70] = -np.inf, np.inf, -np.inf
    res = torch.empty((n, 1, dim), device="cuda", dtype=torch.bfloat16 if out == "bf16" else torch.float32)
    say("packed infinities", dtype, out)
    gpu.packed_attention(q, k, v, res)
    got = host(res)[:, 0]
    assert (got[:, 9] == -np.inf).all()
    assert np.isfinite(got[:7, 70]).all() and (got[7:11, 70] == np.inf).all() and np.isnan(got[11:, 70]).all()
    assert np.isfinite(np.delete(got, [9, 70], 1)).all()
