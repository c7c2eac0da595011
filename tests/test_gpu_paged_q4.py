"""The paged cache of 4-bit codes on the GPU: append against the exact codes, read-back, and decode against float64."""
import numpy as np
import pytest

from gpu_util import dev_bf16, dev_f32, host, say
from oracle import oracle as O
from paged_q4_util import BLOCK, CacheQ4, border_distance, encode64, scored64, unpacked, values64
from paged_util import normed, rounded, turn

pytestmark = pytest.mark.gpu
DIMS = [64, 96, 128, 192, 256]


def dev(x, dtype):
    return dev_bf16(O.pack_bf16(x)) if dtype == "bf16" else dev_f32(x)


def rows_of(cache, new, dtype, seed, behind=0, size=1.0):
    shape = (sum(new) + behind, cache.kv, cache.dim)
    return [rounded(size * O.fill_normal(shape, seed, n), dtype) for n in "kv"]


def starts_of(new):
    import torch
    return torch.tensor([0] + list(new), dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


def appended(gpu, cache, new, k, v, dtype, starts=True, **how):
    """the pool before and after an append: lists of four host arrays"""
    import torch
    pools = cache.device()
    before = [t.cpu().numpy().copy() for t in pools[:4]]
    gpu.paged_append_q4(dev(k, dtype), dev(v, dtype), *pools, starts=starts_of(new) if starts else None, **how)
    torch.cuda.synchronize()
    return before, [t.cpu().numpy() for t in pools[:4]], pools


def check_pool(cache, new, k, v, before, after, off_border=0.0):
    """every new row holds its codes and scales, every other row what it held"""
    untouched = np.ones(before[0].shape[:3], bool)
    first = 0
    for b, n in enumerate(new):
        p = np.arange(cache.lengths[b] - n, cache.lengths[b])
        at = cache.table[b][p // cache.page], slice(None), p % cache.page
        untouched[at] = False
        for i, x in ((0, k), (2, v)):
            x = x[first:first + n]
            codes, scales = encode64(x)
            got, held = unpacked(after[i][at]), after[i + 1][at].astype(np.float64)
            np.testing.assert_array_equal(held, scales)
            clear = border_distance(np.where(np.isfinite(x), x, 0.0)) >= off_border
            np.testing.assert_array_equal(got[clear], codes[clear])
            assert np.abs(got.astype(int) - codes).max(initial=0) <= 1
        first += n
    for was, now in zip(before, after):
        assert np.array_equal(was[untouched], now[untouched], equal_nan=was.dtype == np.float16)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["head", "position"])
def test_append_writes_the_codes_of_its_rows(gpu, dim, dtype, kind):
    new = [3, 1, 0, 17, 40]
    cache = CacheQ4([5, 1, 0, 17, 90], 3, 7, dim, 11, kind)
    k, v = rows_of(cache, new, dtype, 5, behind=2)
    say("append_q4", dim, dtype, kind)
    check_pool(cache, new, k, v, *appended(gpu, cache, new, k, v, dtype)[:2])


def test_append_of_one_token_each(gpu):
    cache = CacheQ4([5, 1, 33, 64], 2, 16, 128, 12)
    k, v = rows_of(cache, [1] * 4, "bf16", 6)
    say("append_q4 without starts")
    check_pool(cache, [1] * 4, k, v, *appended(gpu, cache, [1] * 4, k, v, "bf16", starts=False)[:2])


def special_rows(dim):
    """rows that stand on borders: ties between codes and of scales, zeros, the least and the largest"""
    r = np.random.default_rng(3)
    rows = []
    for s in (2.0 ** -24, 3 * 2.0 ** -24, 129 * 2.0 ** -24, 255 * 2.0 ** -20, 1.0, 129 / 128, 255 / 64, 1360.0, 2720.0):
        x = (r.integers(-14, 15, dim) / 2.0) * s                      # every tie of the code
        x[::BLOCK] = 7 * s
        rows.append(x)
        rows.append(-x)
    rows += [np.zeros(dim), -np.zeros(dim), np.full(dim, 1e-45), np.full(dim, 1e-9), np.full(dim, 3.3e38),
             np.full(dim, 19040.0), np.full(dim, 19041.0), r.normal(size=dim) * 1e30]
    x = r.normal(size=dim)
    for bad in (np.nan, np.inf, -np.inf):
        y = x.copy()
        y[5] = bad
        rows.append(y)
    rows.append(7 * np.nextafter(np.float32(1.0), np.float32(2.0)) * np.ones(dim))       # just past a scale
    rows.append(7 * np.nextafter(np.float32(1.0), np.float32(0.0)) * np.ones(dim))
    return np.array(rows, np.float32)


@pytest.mark.parametrize("dim", [64, 96, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_on_the_borders(gpu, dim, dtype):
    x = rounded(special_rows(dim), dtype)[:, None]
    cache = CacheQ4([len(x)], 1, 8, dim, 4)
    say("append_q4 borders", dim, dtype)
    check_pool(cache, [len(x)], x, x, *appended(gpu, cache, [len(x)], x, x, dtype)[:2])


@pytest.mark.parametrize("dim,rot,interleaved", [(64, 64, False), (96, 40, True), (128, 128, False), (128, 50, False),
                                                 (192, 192, True), (256, 128, False)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_norms_and_turns_the_exact_keys(gpu, dim, rot, interleaved, norm):
    """the codes of the keys in float64; a border nearer than 1e-9 of a scale may fall either way"""
    new, dtype = [2, 30, 5], "bf16"
    cache = CacheQ4([100000, 31, 7], 2, 4096, dim, 13, "position", spare=1, fill=False)
    k, v = rows_of(cache, new, dtype, 7)
    gamma = O.fill_uniform((dim,), 9, "g", 0.5, 1.5) if norm else None
    freqs = (1e4 ** -(np.arange(rot // 2) / (rot // 2))).astype(np.float32)
    say("append_q4 norm and turn", dim, rot, interleaved, norm)
    before, after, _ = appended(gpu, cache, new, k, v, dtype, k_norm=None if gamma is None else dev_f32(gamma),
                                norm_offset=0.25, freqs=dev_f32(freqs), interleaved=interleaved, amplitude=1.25)
    at = np.concatenate([np.arange(n - m, n) for n, m in zip(cache.lengths, new)])
    exact = turn(normed(k, gamma, float(np.float32(1e-6)), 0.25), at, freqs, interleaved, 1.25)
    check_pool(cache, new, exact, v, before, after, off_border=1e-9)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_read_gives_what_the_codes_stand_for(gpu, dim, dtype):
    import torch
    lengths, new = [40, 0, 9, 3], [40, 0, 4, 3]
    cache = CacheQ4(lengths, 3, 10, dim, 21, "position")
    first, behind = 2, 3
    total = first + sum(new) + behind
    wide = torch.full((total, 2, 3 * dim + 4), 7.0, device="cuda", dtype=torch.bfloat16 if dtype == "bf16" else torch.float32)
    k, v = (wide[:, i, :3 * dim].unflatten(-1, (3, dim)) for i in (0, 1))
    starts = starts_of(new) + first
    say("read_q4", dim, dtype)
    gpu.paged_read_q4(k, v, *cache.device(), starts=starts)
    got = host(wide)
    assert (got[:first] == 7).all() and (got[total - behind:] == 7).all() and (got[:, :, 3 * dim:] == 7).all()
    at = first
    for b, n in enumerate(new):
        for i, x in enumerate(cache.rows(b)):
            want = rounded(x[lengths[b] - n:], dtype).reshape(n, 3 * dim)
            np.testing.assert_array_equal(got[at:at + n, i, :3 * dim], want)
        at += n


def test_read_of_places_that_are_none(gpu):
    """a page outside the pool and a length below the new tokens read as NaN, neighbours as they are"""
    import torch
    cache = CacheQ4([20, 20, 2], 2, 8, 64, 22)
    cache.table[1, 1] = cache.pages
    out = [torch.zeros((44, 2, 64), device="cuda") for _ in "kv"]
    say("read_q4 bad places")
    gpu.paged_read_q4(*out, *cache.device(), starts=starts_of([20, 20, 4]))
    for i, x in enumerate(out):
        x = host(x)
        np.testing.assert_array_equal(x[:20], cache.rows(0)[i])
        np.testing.assert_array_equal(np.isnan(x[20:40]).all((1, 2)), (np.arange(20) // 8) == 1)
        assert np.isnan(x[40:42]).all()
        np.testing.assert_array_equal(x[42:], cache.rows(2)[i])


def decoded(gpu, cache, q, dtype, **how):
    import torch
    out = torch.full((len(cache.lengths), q.shape[1], cache.dim), 5.0, device="cuda")
    gpu.paged_decode_q4(dev(q, dtype), out, *cache.device(), **how)
    return host(out)


def check_decode(cache, got, q, **how):
    for b, n in enumerate(cache.lengths):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        keys, values = cache.rows(b)
        # two terms of 11 bits: 2^-22 of a value
        want, bound = scored64(q[b], keys, values, n - 1, terms=2, product=4.0, **how)
        assert (np.abs(got[b] - want) <= bound).all(), (b, n, np.abs(got[b] - want).max(), (np.abs(got[b] - want) / bound).max())


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("heads,kv", [(12, 12), (8, 2), (16, 1), (24, 1), (5, 5)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_against_64_bits(gpu, dim, heads, kv, dtype):
    cache = CacheQ4([1, 0, 63, 64, 65, 130, 777], kv, 9, dim, 31)
    q = rounded(O.fill_normal((7, heads, dim), 8, "q"), dtype)
    say("decode_q4", dim, heads, kv, dtype)
    check_decode(cache, decoded(gpu, cache, q, dtype), q)


@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("cap,biased,window", [(30.0, False, 0), (2.0, False, 0), (0.0, True, 0), (20.0, True, 100),
                                               (0.0, False, 1), (0.0, True, 64)])
def test_decode_capped_biased_windowed(gpu, dim, cap, biased, window):
    cache = CacheQ4([1, 200, 33, 1500], 2, 16, dim, 32, "position")
    q = 3 * O.fill_normal((4, 6, dim), 8, "q")
    slopes = (2.0 ** -np.arange(1, 7)).astype(np.float32) if biased else None
    say("decode_q4 forms", dim, cap, biased, window)
    got = decoded(gpu, cache, q, "f32", cap=cap, slopes=None if slopes is None else dev_f32(slopes), window=window)
    check_decode(cache, got, q, cap=cap, slopes=slopes, window=window)


@pytest.mark.parametrize("dim,rot,interleaved", [(64, 64, False), (96, 96, False), (128, 128, False), (128, 30, True),
                                                 (192, 100, False), (256, 256, False)])
def test_decode_norms_and_turns_q(gpu, dim, rot, interleaved):
    cache = CacheQ4([300, 4, 70], 2, 32, dim, 33)
    q = O.fill_normal((3, 8, dim), 9, "q")
    gamma = O.fill_uniform((dim,), 9, "g", 0.5, 1.5)
    freqs = (1e4 ** -(np.arange(rot // 2) / (rot // 2))).astype(np.float32)
    say("decode_q4 norm and turn", dim, rot, interleaved)
    got = decoded(gpu, cache, q, "f32", q_norm=dev_f32(gamma), freqs=dev_f32(freqs), interleaved=interleaved,
                  norm_offset=0.5)
    check_decode(cache, got, q, gamma=gamma, freqs=freqs, interleaved=interleaved, offset=0.5)


@pytest.mark.parametrize("size,qsize", [(1e-6, 1.0), (2000.0, 1e-3), (1.0, 1e-30), (1e-4, 1e4), (3000.0, 1e30)])
def test_decode_of_small_and_large_values(gpu, size, qsize):
    """scales down to fp16's least and up to the largest, queries of any size (huge ones pick one key)"""
    cache = CacheQ4([130, 20], 2, 16, 128, 34, size=size)
    q = (qsize * O.fill_normal((2, 4, 128), 8, "q")).astype(np.float32)
    say("decode_q4 sizes", size, qsize)
    got = decoded(gpu, cache, q, "f32")
    assert np.isfinite(got).all()
    if qsize < 1e30:
        check_decode(cache, got, q)
    else:
        for b in range(2):
            keys, values = cache.rows(b)
            for h in range(4):
                best = (keys[:, h // 2] @ q[b, h].astype(np.float64)).argmax()
                np.testing.assert_allclose(got[b, h], values[best, h // 2], rtol=1e-6, atol=0)


def test_decode_of_lengths_and_pages_that_cannot_be(gpu):
    cache = CacheQ4([50, 40, 30, 0], 2, 8, 64, 35)
    q = O.fill_normal((4, 4, 64), 8, "q")
    lengths = list(cache.lengths)
    cache.table[1, 2] = cache.pages + 5
    cache.lengths[2] = 57                  # past max_length
    say("decode_q4 bad pages")
    got = decoded(gpu, cache, q, "f32", max_length=56)
    assert np.isnan(got[1]).all() and np.isnan(got[2]).all() and (got[3] == 0).all()
    cache.lengths = lengths[:1]
    check_decode(cache, got[:1], q)


def test_decode_gates_its_output(gpu):
    cache = CacheQ4([77, 5], 1, 16, 96, 36)
    q = O.fill_normal((2, 3, 192), 8, "q")
    say("decode_q4 gate")
    got = decoded(gpu, cache, q, "f32", output_gate=True)
    plain = decoded(gpu, cache, np.ascontiguousarray(q[..., :96]), "f32")
    gate = 1 / (1 + np.exp(-q[..., 96:].astype(np.float64)))
    # the gate's exponential, sum, quotient and product
    np.testing.assert_allclose(got, plain * gate, rtol=8 * 2.0 ** -24, atol=1e-30)


def test_decode_of_one_long_sequence_among_short_ones(gpu):
    """records of many workgroups, joined in the launch and by the second one"""
    for batch, length in ((1, 40000), (64, 9000)):
        cache = CacheQ4([length] + [3] * (batch - 1), 1, 64, 64, 37)
        q = O.fill_normal((batch, 4, 64), 8, "q")
        say("decode_q4 long", batch, length)
        check_decode(cache, decoded(gpu, cache, q, "f32"), q)


def test_a_captured_decode_follows_the_lengths(gpu):
    """append and decode captured once, replayed with new tokens and lengths between eager work"""
    import torch
    cache = CacheQ4([40, 3, 64], 2, 16, 128, 38, width=8, spare=16)
    used = {p for b, n in enumerate(cache.lengths) for p in cache.table[b, :-(-n // 16)].tolist()}
    free = [p for p in range(cache.pages) if p not in used]
    for b, n in enumerate(cache.lengths):            # every place of the table has a page
        for slot in range(-(-n // 16), 8):
            cache.table[b, slot] = free.pop()
    pools = cache.device()
    kv = torch.randn((3, 4, 128), device="cuda", dtype=torch.bfloat16)
    q = torch.randn((3, 4, 128), device="cuda")
    out = torch.empty((3, 4, 128), device="cuda")
    say("decode_q4 captured")
    work = gpu.paged_decode_q4_workspace(q, out, *pools)

    def step():
        gpu.paged_append_q4(kv[:, :2], kv[:, 2:], *pools)
        gpu.paged_decode_q4(q, out, *pools, workspace=work)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        kv.normal_()
        q.normal_()
        pools[-1].add_(1)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        again = torch.empty_like(out)
        gpu.paged_decode_q4(q, again, *pools)
        torch.cuda.synchronize()
        assert torch.isfinite(got).all() and torch.equal(got, again), i
        read = torch.empty((3, 2, 128), device="cuda"), torch.empty((3, 2, 128), device="cuda")
        gpu.paged_read_q4(*read, *pools)
        for x, rows in zip(read, (kv[:, :2], kv[:, 2:])):
            np.testing.assert_array_equal(host(x), values64(*encode64(host(rows))))


def test_decode_on_two_streams(gpu):
    """calls of two streams at once, each with the backend's own scratch"""
    import torch
    cache = CacheQ4([3000, 500, 0, 1200], 2, 16, 128, 39)
    pools = cache.device()
    qs = [O.fill_normal((4, 8, 128), 40 + i, "q") for i in range(2)]
    outs = [torch.empty((4, 8, 128), device="cuda") for _ in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    devs = [dev_f32(q) for q in qs]
    torch.cuda.synchronize()
    say("decode_q4 two streams")
    for _ in range(20):
        for q, out, stream in zip(devs, outs, streams):
            with torch.cuda.stream(stream):
                gpu.paged_decode_q4(q, out, *pools)
    torch.cuda.synchronize()
    for q, out in zip(qs, outs):
        check_decode(cache, host(out), q)
