"""Values that are not finite, among the documents of a packed attention: as the weighted sum has it, each reaches its
own channel of the tokens that see its row, whichever tiles and splits the rows fall into."""
import numpy as np
import pytest

from gpu_util import host, say
from oracle import oracle as O
from packed_util import document64
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


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
def test_scores_that_are_all_minus_infinity(gpu, dim, dtype, out):
    """no weight is left: NaN, in one call's documents, behind split keys and in the decode alike; a key whose score
    is -infinity leaves the weights to the others; a token that sees nothing gets zeros"""
    import torch
    new, sizes, kv = [40, 3, 9], [40, 3000, 4], 1
    starts, keys = np.cumsum([0] + new), np.cumsum([0] + sizes)
    q, k, v = (rounded(O.fill_normal((m, h, dim), 33, s), dtype)
               for m, h, s in ((starts[-1], 2, "q"), (keys[-1], kv, "k"), (keys[-1], kv, "v")))
    q[..., 0] = np.abs(q[..., 0]) + 1
    q = rounded(q, dtype)
    k[0, 0, 0] = -np.inf                   # of the first document, its first key
    k[keys[1]:keys[2], 0, 0] = -np.inf     # of the second, all; the third has five tokens before its keys
    res = torch.full((starts[-1], 2, dim), 3.0, device="cuda", dtype=torch.bfloat16 if out == "bf16" else torch.float32)
    tensors = dev(q, dtype), dev(k, dtype), dev(v, dtype), res
    for alone in (False, True):
        say("packed no weights", dim, dtype, out, alone)
        # many documents' keys are few on average, the second one's by themselves enough to be split
        for b in [slice(i, i + 1) for i in range(3)] if alone else [slice(0, 3)]:
            at, ka = slice(starts[b.start], starts[b.stop]), slice(keys[b.start], keys[b.stop])
            call = tensors[0][at], tensors[1][ka], tensors[2][ka], res[at]
            how = dict(starts=vector((starts[b.start:b.stop + 1] - starts[b.start]).tolist()),
                       key_starts=vector((keys[b.start:b.stop + 1] - keys[b.start]).tolist()))
            assert (gpu.packed_attention_workspace(*call, **how).numel() > 0) == (alone and b.start == 1)
            gpu.packed_attention(*call, **how)
        got = host(res)
        assert np.isnan(got[0]).all() and np.isnan(got[40:43]).all()
        assert (got[43:48] == 0).all() and np.isfinite(got[48:]).all()
        want, bound = document64(q[1:40], k[1:40], v[1:40], dtype, out)
        assert (np.abs(got[1:40] - want) <= bound).all()
        res.fill_(3.0)
    pages = dev(k[keys[1]:keys[1] + 16], "bf16").reshape(1, 1, 16, dim)
    one = torch.zeros((1, 2, dim), device="cuda")
    gpu.paged_decode(dev(q[:1], "f32"), one, pages, pages.nan_to_num(neginf=0.0), vector([[0]]), vector([16]))
    assert np.isnan(host(one)).all()
