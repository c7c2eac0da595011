"""Packed attention and the 4-bit cache where their index arithmetic and their scratch
can go wrong: offsets past 32 bits, wide strides, strided pools, streams, repeats."""
import numpy as np
import pytest

from gpu_util import dev_f32, host, say
from oracle import oracle as O
from packed_util import document64
from paged_q4_util import CacheQ4, encode64, scored64, unpacked, values64
from paged_util import rounded
from test_gpu_packed import dev, starts_of, vector

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stride,keys,first", [(1 << 24, 24, 0), (1 << 20, 2600, 2500)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_keys_far_apart(gpu, stride, keys, first, dtype):
    """a tile whose rows are gigabytes apart, and documents past 4 GB of keys"""
    import torch
    kind, D = (torch.bfloat16, 64) if dtype == "bf16" else (torch.float32, 64)
    if dtype == "f32":
        stride //= 2
    say("packed far keys", stride, keys, dtype)
    room = torch.empty(keys * stride + D, dtype=kind, device="cuda")
    k = room.as_strided((keys, 1, D), (stride, D, 1))
    v = room[D:].as_strided((keys, 1, D), (stride, D, 1)) if stride >= 2 * D else None
    n = keys - first
    rows = {s: rounded(O.fill_normal((n, 1, D), 3, s), dtype) for s in "kv"}
    k.fill_(float("nan"))
    v.fill_(float("nan"))
    k[first:], v[first:] = dev(rows["k"], dtype), dev(rows["v"], dtype)
    q = rounded(O.fill_normal((n, 2, D), 3, "q"), dtype)
    out = torch.empty((n, 2, D), device="cuda")
    gpu.packed_attention(dev(q, dtype), k, v, out, starts=vector([0, 0, n]), key_starts=vector([0, first, keys]))
    want, bound = document64(q, rows["k"], rows["v"], dtype, "f32")
    got = host(out)
    del room, k, v
    assert (np.abs(got - want) <= bound).all()


def test_pages_past_4_gb(gpu):
    """codes of more than 4 GB: append, read-back and decode at the pool's end"""
    import torch
    D, size, pages = 256, 16, (1 << 32) // (256 // 2 * 16) + 100
    say("q4 far pages", pages)
    codes = [torch.zeros((pages, 1, size, D // 2), dtype=torch.uint8, device="cuda") for _ in "kv"]
    scales = [torch.zeros((pages, 1, size, D // 32), dtype=torch.float16, device="cuda") for _ in "kv"]
    table = vector(list(range(pages - 1, pages - 9, -1))).reshape(1, 8)
    lengths = vector([120])
    k, v = (O.fill_normal((120, 1, D), 4, s) for s in "kv")
    pools = codes[0], scales[0], codes[1], scales[1], table, lengths
    gpu.paged_append_q4(dev_f32(k), dev_f32(v), *pools, starts=vector([0, 120]))
    read = [torch.empty((120, 1, D), device="cuda") for _ in "kv"]
    gpu.paged_read_q4(*read, *pools, starts=vector([0, 120]))
    for got, x in zip(read, (k, v)):
        np.testing.assert_array_equal(host(got), values64(*encode64(x)))
    q, out = O.fill_normal((1, 4, D), 4, "q"), torch.empty((1, 4, D), device="cuda")
    gpu.paged_decode_q4(dev_f32(q), out, *pools)
    want, bound = scored64(q[0], host(read[0]).astype(np.float64), host(read[1]).astype(np.float64), 119, terms=2, product=4.0)
    assert (np.abs(host(out)[0] - want) <= bound).all()
    assert int(codes[0][0].sum()) == 0 and int(codes[0][(1 << 32) // (D // 2 * size) // 2].sum()) == 0


@pytest.mark.parametrize("dim", [64, 96, 256])
def test_pools_of_other_strides(gpu, dim):
    """keys and values as the halves of one buffer of pages"""
    import torch
    cache = CacheQ4([50, 7, 0, 33], 2, 8, dim, 61)
    dense = cache.device()
    both = [torch.zeros((cache.pages, 2, 2, 8, dim // 2), dtype=torch.uint8, device="cuda"),
            torch.zeros((cache.pages, 2, 2, 8, dim // 32), dtype=torch.float16, device="cuda")]
    pools = [t[:, i] for i in (0, 1) for t in both]
    for t, x in zip(pools, dense[:4]):
        t.copy_(x)
    q = dev_f32(O.fill_normal((4, 4, dim), 8, "q"))
    a, b = torch.empty((4, 4, dim), device="cuda"), torch.empty((4, 4, dim), device="cuda")
    say("q4 strided pools", dim)
    gpu.paged_decode_q4(q, a, *dense)
    gpu.paged_decode_q4(q, b, *pools, *dense[4:])
    new = O.fill_normal((4, 4, dim), 9, "n")
    for p in (dense[:4], pools):
        gpu.paged_append_q4(dev_f32(new[:, :2]), dev_f32(new[:, 2:]), *p, *dense[4:])
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    for x, y in zip(dense[:4], pools):
        np.testing.assert_array_equal(x.cpu().numpy(), y.cpu().numpy())


@pytest.mark.parametrize("page", [1, 5, 64, 1000])
def test_pages_of_any_size(gpu, page):
    import torch
    cache = CacheQ4([1, 64, 129, 200], 2, page, 128, 62, "position")
    q, out = O.fill_normal((4, 4, 128), 8, "q"), torch.empty((4, 4, 128), device="cuda")
    say("q4 page size", page)
    gpu.paged_decode_q4(dev_f32(q), out, *cache.device())
    for b, n in enumerate(cache.lengths):
        want, bound = scored64(q[b], *cache.rows(b), n - 1, terms=2, product=4.0)
        assert (np.abs(host(out)[b] - want) <= bound).all(), b


def test_a_batch_of_empty_places(gpu):
    import torch
    cache = CacheQ4([0, 0, 0], 2, 16, 64, 63)
    out = torch.ones((3, 4, 64), device="cuda")
    say("q4 empty batch")
    gpu.paged_decode_q4(dev_f32(O.fill_normal((3, 4, 64), 8, "q")), out, *cache.device())
    assert (host(out) == 0).all()
    x = torch.ones((5, 4, 64), device="cuda", dtype=torch.bfloat16)
    res = torch.full_like(x, 3.0)
    gpu.packed_attention(x, x[:, :2].contiguous(), x[:, :2].contiguous(), res, starts=vector([2, 2, 2]))
    assert (host(res) == 3).all()


def test_results_do_not_depend_on_timing(gpu):
    """split keys and joined records: the same bits every time, beside other work and on two streams"""
    import torch
    H, KV, D = 8, 2, 128
    new, past = [3, 17, 1], [5000, 900, 12000]
    lengths = [a + b for a, b in zip(new, past)]
    q = torch.randn((sum(new), H, D), device="cuda", dtype=torch.bfloat16)
    k, v = (torch.randn((sum(lengths), KV, D), device="cuda", dtype=torch.bfloat16) for _ in "kv")
    how = dict(starts=vector(starts_of(new)), key_starts=vector(starts_of(lengths)))
    cache = CacheQ4([9000, 3, 400], 2, 16, 128, 64)
    pools, q4 = cache.device(), torch.randn((3, H, D), device="cuda")
    first, first4 = torch.empty((sum(new), H, D), device="cuda"), torch.empty((3, H, D), device="cuda")
    say("repeats")
    gpu.packed_attention(q, k, v, first, **how)
    gpu.paged_decode_q4(q4, first4, *pools)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            outs.append((torch.empty_like(first), torch.empty_like(first4)))
            gpu.packed_attention(q, k, v, outs[-1][0], **how)
            gpu.paged_decode_q4(q4, outs[-1][1], *pools)
    torch.cuda.synchronize()
    for a, b in outs:
        assert torch.equal(a, first) and torch.equal(b, first4)


@pytest.mark.parametrize("dim", [128, 192, 256])
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
def test_long_documents(gpu, dim, dtype, out):
    """many tiles a workgroup, its waves at different ends of a window"""
    import torch
    n, H, KV = 1500, 3, 1
    q, k, v = (rounded(O.fill_normal((n, h, dim), 12, s), dtype) for h, s in ((H, "q"), (KV, "k"), (KV, "v")))
    slopes = np.array([0.3, 0.01, 0.0], np.float32)
    res = torch.empty((n, H, dim), device="cuda", dtype=torch.bfloat16 if out == "bf16" else torch.float32)
    say("packed long", dim, dtype, out)
    for how in (dict(), dict(window=333, prefix=[700], cap=30.0)):
        args = dict(how, prefix=vector(how["prefix"])) if "prefix" in how else how
        gpu.packed_attention(dev(q, dtype), dev(k, dtype), dev(v, dtype), res, starts=vector([0, n]),
                             slopes=dev_f32(slopes), **args)
        ref = dict(how, prefix=how["prefix"][0]) if "prefix" in how else how
        want, bound = document64(q, k, v, dtype, out, slopes=slopes, **ref)
        assert (np.abs(host(res) - want) <= bound).all()


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("new,past,how", [
    (200, 0, {}), (200, 0, dict(window=45)), (200, 0, dict(prefix=90)), (150, 0, dict(prefix=150, window=20)),
    (21, 1500, {}), (21, 1500, dict(window=700)),
])
def test_rows_that_are_not_finite_reach_those_that_see_them(gpu, dim, dtype, out, new, past, how):
    """a key or value with NaN or an infinity: NaN (or infinite) for the tokens and heads that
    see it; the others' results are those of finite rows, to the bit"""
    import torch
    n, H, KV = new + past, 4, 2
    q, k, v = (dev(rounded(O.fill_normal((m, h, dim), 21, s), dtype), dtype)
               for m, h, s in ((new, H, "q"), (n, KV, "k"), (n, KV, "v")))
    window, prefix = how.get("window", 0), how.get("prefix", 0)
    args = dict(starts=vector([0, new]), key_starts=vector([0, n]), window=window)
    if prefix:
        args["prefix"] = vector([prefix])
    plain, got = (torch.zeros((new, H, dim), device="cuda", dtype=torch.bfloat16 if out == "bf16" else torch.float32) for _ in "ab")
    say("packed wild", dim, dtype, out, new, past, how)
    gpu.packed_attention(q, k, v, plain, **args)
    i, j = np.arange(past, n)[:, None], np.arange(n)[None]
    sees = ((j <= i) | (j < prefix)) & ((window == 0) | (i - j < window))
    for where, at, bad in (("v", n - 1, np.nan), ("v", n - 17, np.inf), ("k", n - 9, np.nan), ("v", past + 3, -np.inf), ("v", n // 2, np.nan)):
        kk, vv = k.clone(), v.clone()
        (kk if where == "k" else vv)[at, 1, dim // 2 + 5] = bad
        gpu.packed_attention(q, kk, vv, got, **args)
        a, b = host(plain), host(got)
        np.testing.assert_array_equal(a[:, :2], b[:, :2])
        np.testing.assert_array_equal(a[~sees[:, at], 2:], b[~sees[:, at], 2:])
        assert not np.isfinite(b[sees[:, at], 2:]).all(-1).any()


def test_capped_scores_beside_rows_that_are_not_finite(gpu):
    import torch
    n, H, dim = 130, 4, 128
    q, k, v = (rounded(O.fill_normal((n, h, dim), 22, s), "bf16") for h, s in ((H, "q"), (1, "k"), (1, "v")))
    slopes = np.array([0.3, 0.01, 0.0, 1.0], np.float32)
    kk, vv = dev(k, "bf16"), dev(v, "bf16")
    kk[100, 0, 7], vv[101, 0, 0] = np.inf, np.nan
    out = torch.empty((n, H, dim), device="cuda", dtype=torch.bfloat16)
    say("packed wild, capped")
    gpu.packed_attention(dev(q, "bf16"), kk, vv, out, cap=20.0, slopes=dev_f32(slopes))
    want, bound = document64(q[:100], k[:100], v[:100], "bf16", "bf16", slopes=slopes, cap=20.0)
    assert (np.abs(host(out)[:100] - want) <= bound).all()


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("cap", [1e-6, 1e-3, 1.0, 300.0, 2e4, 1e6])
def test_caps_of_any_size(gpu, dtype, out, cap):
    """scores of 0, far below the cap, about it and past it, whatever the cap"""
    import torch
    n, H, dim = 200, 4, 128
    q, k, v = (O.fill_normal((n, h, dim), 23, s) for h, s in ((H, "q"), (1, "k"), (1, "v")))
    q[::5] *= 1e-4
    q[1::5] *= 30.0
    q[2::5] *= min(cap, 1e3)
    q[7] = 0.0
    q, k, v = (rounded(x, dtype) for x in (q, k, v))
    res = torch.empty((n, H, dim), device="cuda", dtype=torch.bfloat16 if out == "bf16" else torch.float32)
    say("packed cap", cap, dtype, out)
    gpu.packed_attention(dev(q, dtype), dev(k, dtype), dev(v, dtype), res, cap=cap)
    want, bound = document64(q, k, v, dtype, out, cap=cap)
    assert (np.abs(host(res) - want) <= bound).all()


@pytest.mark.parametrize("cap", [1e-6, 1e-3, 300.0, 1e6])
def test_decode_caps_of_any_size(gpu, cap):
    import torch
    cache = CacheQ4([300, 64, 1], 1, 16, 128, 24)
    q, out = O.fill_normal((3, 4, 128), 24, "q"), torch.empty((3, 4, 128), device="cuda")
    q[:, 0] = 0.0
    q[:, 1] *= min(cap, 30.0)
    say("q4 cap", cap)
    gpu.paged_decode_q4(dev_f32(q), out, *cache.device(), cap=cap)
    for b, n in enumerate(cache.lengths):
        want, bound = scored64(q[b], *cache.rows(b), n - 1, cap=cap, terms=2, product=4.0)
        assert (np.abs(host(out)[b] - want) <= bound).all(), b
