"""GPU parity of the paged cache against float64: aigpu_paged_append and
aigpu_paged_decode each by itself, and together as a serving loop uses them.
The pools hold NaN wherever no position lies (tests/paged_util.py)."""
import numpy as np
import pytest

from common import gammas
from gpu_util import dev_f32, dev_u32, host, host_bits, say
from oracle import oracle as O
from paged_util import HALF_STEP, NORM_STEPS, TURN_STEPS, U, Cache, decode64, normed, pair_sizes, rounded, turn

pytestmark = pytest.mark.gpu


def _dev(x, dtype):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda().to(torch.bfloat16 if dtype == "bf16" else torch.float32)


def _options(dim, seed, norm, rot, interleaved=False, amplitude=1.0):
    return dict(gamma=gammas(dim, seed, "g") if norm else None,
                freqs=O.rotary_frequencies(rot, 1e6) if rot else None, interleaved=interleaved, amplitude=amplitude)


def _decode(gpu, cache, q, dtype, opt, device=None, **kw):
    """the GPU's answer for q [batch][heads][width] as numpy"""
    import torch
    keys, values, table, lengths = device or cache.device()
    out = torch.full((q.shape[0], q.shape[1], cache.dim), 7.0, device="cuda")
    t = q if isinstance(q, torch.Tensor) else _dev(q, dtype)
    say("paged decode", dict(lengths=cache.lengths[:8], batch=len(cache.lengths), heads=q.shape[1], kv=cache.kv,
                             dim=cache.dim, page=cache.page, kind=cache.kind, dtype=dtype), kw)
    gpu.paged_decode(t, out, keys, values, table, lengths, q_norm=None if opt["gamma"] is None else dev_f32(opt["gamma"]),
                     freqs=None if opt["freqs"] is None else dev_f32(opt["freqs"]), interleaved=opt["interleaved"],
                     amplitude=opt["amplitude"], **kw)
    return host(out)


def _check_decode(got, cache, q, opt, window=0, scale=0.0, skip=()):
    for b, n in enumerate(cache.lengths):
        if b in skip:
            continue
        if n == 0:
            assert (got[b] == 0).all()
            continue
        k, v = cache.rows(b)
        want, bound = decode64(q[b][:, :cache.dim], k, v, n - 1, window=window, scale=scale, **opt)
        err = np.abs(got[b] - want)
        assert (err <= bound).all(), (b, n, (err / bound).max())


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("heads,kv", [(1, 1), (12, 12), (16, 8), (15, 3), (32, 4), (16, 1), (40, 2)])
def test_decode_heads(gpu, dim, heads, kv):
    opt = _options(dim, 1, True, dim)
    cache = Cache([300, 0, 1, 33, 700], kv, 16, dim, dim + heads)
    q = rounded(2 * O.fill_normal((5, heads, dim), 2, "q"), "bf16")
    _check_decode(_decode(gpu, cache, q, "bf16", opt), cache, q, opt)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 31, 32, 33, 64, 100, 256, 1000])
@pytest.mark.parametrize("kind", ["head", "position"])
def test_decode_pages(gpu, page, kind):
    opt = _options(128, 3, False, 128)
    cache = Cache([1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 999, 1000, 1001], 2, page, 128, page, kind)
    q = rounded(3 * O.fill_normal((15, 8, 128), 4, "q"), "f32")
    _check_decode(_decode(gpu, cache, q, "f32", opt), cache, q, opt)


@pytest.mark.parametrize("window", [1, 7, 32, 100, 1000, 5000])
def test_decode_window(gpu, window):
    opt = _options(64, 5, True, 32, True)
    cache = Cache([1200, 5, 299, 0, 1000, 1001, 4000], 2, 24, 64, 6)
    q = rounded(2 * O.fill_normal((7, 8, 64), 7, "q"), "bf16")
    _check_decode(_decode(gpu, cache, q, "bf16", opt, window=window), cache, q, opt, window=window)


@pytest.mark.parametrize("norm,rot,interleaved,amplitude,dtype",
                         [(False, 0, False, 1.0, "f32"), (True, 0, False, 1.0, "bf16"), (True, 128, True, 1.1, "f32"),
                          (False, 14, False, 0.5, "bf16"), (True, 2, True, 1.0, "f32"), (True, 126, False, 2.0, "f32")])
def test_decode_query_forms(gpu, norm, rot, interleaved, amplitude, dtype):
    opt = _options(128, 8, norm, rot, interleaved, amplitude)
    cache = Cache([90, 2000], 2, 16, 128, 9)
    q = rounded(O.fill_normal((2, 8, 128), 10, "q"), dtype)
    _check_decode(_decode(gpu, cache, q, dtype, opt), cache, q, opt)


def test_decode_scale_norm_offset_and_strided_queries(gpu):
    """q as the middle of wider rows; the norm's offset and a scale of one's own"""
    import torch
    opt = dict(_options(128, 11, True, 64), eps=1e-3, offset=1.0)
    cache = Cache([77, 640, 3], 2, 16, 128, 12)
    rows = rounded(O.fill_normal((3, 24, 128), 13, "q"), "bf16")
    wide = _dev(rows, "bf16")
    got = _decode(gpu, cache, wide[:, 8:16], "bf16", opt, scale=0.03, eps=1e-3, norm_offset=1.0)
    _check_decode(got, cache, rows[:, 8:16], opt, scale=0.03)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_off_16_bytes(gpu, dtype):
    """queries, keys and values that start on no 16-byte boundary"""
    import torch
    opt = _options(96, 90, True, 40)
    cache = Cache([77, 640, 1], 3, 16, 96, 91)
    flat = rounded(O.fill_normal((3 * 6 * 96 + 1,), 92, "q"), dtype)
    off = _dev(flat, dtype)[1:].view(3, 6, 96)
    assert off.data_ptr() % 16
    q = flat[1:].reshape(3, 6, 96)
    device = cache.device()
    _check_decode(_decode(gpu, cache, off, dtype, opt, device=device), cache, q, opt)
    k, v = off[:, :3], _dev(flat, dtype)[:-1].view(3, 6, 96)[:, 3:]
    gpu.paged_append(k, v, *device)
    keys, values = host(device[0]), host_bits(device[1])
    for b, n in enumerate(cache.lengths):
        at = cache.table[b][(n - 1) // 16], slice(None), (n - 1) % 16
        assert np.array_equal(keys[at], rounded(q[b, :3], "bf16"))
        assert np.array_equal(values[at], O.pack_bf16(flat[:-1].reshape(3, 6, 96)[b, 3:]).reshape(3, 96))


def test_decode_repeats_to_the_bit(gpu):
    """whichever workgroup joins a sequence's parts"""
    opt = _options(128, 93, True, 128)
    cache = Cache([12000, 3, 700, 5000, 64, 1, 8191, 0, 2500], 4, 16, 128, 94)
    q = rounded(O.fill_normal((9, 32, 128), 95, "q"), "bf16")
    device = cache.device()
    first = _decode(gpu, cache, q, "bf16", opt, device=device)
    for _ in range(30):
        assert np.array_equal(_decode(gpu, cache, q, "bf16", opt, device=device), first)


@pytest.mark.parametrize("heads", [8, 40])
def test_decode_output_gate(gpu, heads):
    opt = _options(128, 14, True, 128)
    cache = Cache([50, 3000, 0], 2, 16, 128, 15)
    q = rounded(O.fill_normal((3, heads, 256), 16, "q"), "bf16")
    got = _decode(gpu, cache, q, "bf16", opt, output_gate=True)
    for b, n in enumerate(cache.lengths):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        k, v = cache.rows(b)
        want, bound = decode64(q[b][:, :128], k, v, n - 1, **opt)
        gate = 1 / (1 + np.exp(-q[b][:, 128:].astype(np.float64)))
        err = np.abs(got[b] - want * gate)
        assert (err <= bound * gate + 8 * U * np.abs(want * gate)).all()


@pytest.mark.parametrize("lengths", [[20000], [9000, 1, 12345, 4097], [5] * 300, [i % 90 for i in range(1100)]])
def test_decode_batches(gpu, lengths):
    """one long sequence, ragged ones, many short ones, and more sequences than a launch's plan holds"""
    opt = _options(64, 17, False, 64)
    kv = 1 if len(lengths) > 1000 else 2
    cache = Cache(lengths, kv, 16, 64, 18)
    q = rounded(2 * O.fill_normal((len(lengths), 4, 64), 19, "q"), "f32")
    _check_decode(_decode(gpu, cache, q, "f32", opt, max_length=max(lengths)), cache, q, opt)


def test_decode_finds_one_key_among_many(gpu):
    """a key aligned with q outweighs all others wherever it lies: each position is read once, from its own row"""
    import torch
    n, dim = 1500, 64
    opt = _options(dim, 0, False, 0)
    places = [0, 1, 15, 16, 31, 32, 33, 63, 64, 127, 128, 700, 1023, 1024, 1471, 1472, 1498, 1499]
    cache = Cache([n] * len(places), 1, 24, dim, 20)
    q = rounded(np.sign(O.fill_normal((len(places), 1, dim), 21, "q")), "bf16")
    for b, p in enumerate(places):
        cache.keys[cache.table[b][p // 24], 0, p % 24] = 4 * q[b, 0]
    got = _decode(gpu, cache, q, "bf16", opt)
    _check_decode(got, cache, q, opt)
    for b, p in enumerate(places):
        assert np.abs(got[b, 0] - cache.rows(b)[1][p, 0]).max() < 1e-3    # e^-20 of 1500 others is left


def test_decode_extreme_scores(gpu):
    """scores of +-60000: weights underflow to the one winner, nothing overflows"""
    opt = _options(128, 0, False, 0)
    cache = Cache([400, 37], 1, 16, 128, 22)
    q = rounded(3000 * O.fill_normal((2, 2, 128), 23, "q"), "f32")
    got = _decode(gpu, cache, q, "f32", opt)
    assert np.isfinite(got).all()
    _check_decode(got, cache, q, opt)


def test_decode_bad_places_answer_nan(gpu):
    """a length past max_length, a page outside the pool (inside the attended part, or only before the window), a
    length past the table: NaN for that sequence alone, nothing read outside"""
    opt = _options(128, 0, False, 128)
    cache = Cache([200, 200, 200, 200, 200, 200], 2, 16, 128, 24)
    q = rounded(O.fill_normal((6, 4, 128), 25, "q"), "bf16")
    device = cache.device()
    device[3][1] = 2 ** 31 - 1          # a length past everything
    device[3][2] = -1
    device[2][3, 5] = cache.pages       # one past the pool
    device[2][4, 12] = -1               # its last page
    device[2][5, 0] = -7                # its first
    got = _decode(gpu, cache, q, "bf16", opt, device=device, max_length=200)
    assert np.isnan(got[1:]).all()
    _check_decode(got, cache, q, opt, skip=range(1, 6))
    got = _decode(gpu, cache, q, "bf16", opt, device=device, max_length=199)
    assert np.isnan(got).all()
    got = _decode(gpu, cache, q, "bf16", opt, device=device, max_length=200, window=100)
    assert np.isnan(got[[1, 2, 4]]).all()      # page 5 holds positions 80 to 95, outside the window too
    _check_decode(got, cache, q, opt, window=100, skip=(1, 2, 4))


def test_decode_offsets_past_32_bits(gpu):
    """a pool of more than 2^32 elements whose last pages are in use"""
    import torch
    page, kv, dim = 256, 8, 128
    pages = 2 ** 32 // (page * kv * dim) + 40
    keys = torch.zeros((pages, kv, page, dim), dtype=torch.bfloat16, device="cuda")
    values = torch.zeros_like(keys)
    assert keys.numel() > 2 ** 32
    cache = Cache([9000, 300], kv, page, dim, 26, spare=0)
    small_k, small_v, table, lengths = cache.device()
    keys[pages - cache.pages:] = small_k
    values[pages - cache.pages:] = small_v
    live = table < cache.pages
    table[live] += pages - cache.pages
    opt = _options(dim, 27, True, dim)
    q = rounded(O.fill_normal((2, 16, dim), 28, "q"), "bf16")
    got = _decode(gpu, cache, q, "bf16", opt, device=(keys, values, table, lengths))
    _check_decode(got, cache, q, opt)
    k = rounded(O.fill_normal((2, kv, dim), 29, "k"), "bf16")
    gpu.paged_append(_dev(k, "bf16"), _dev(k, "bf16"), keys, values, table, lengths)
    at = table[0, 8999 // page].item()
    assert np.array_equal(host(values[at, :, 8999 % page].contiguous()), k[0])
    assert int((values[:pages - cache.pages] != 0).sum()) == 0


@pytest.mark.parametrize("dim,kv,dtype,rot,interleaved,norm",
                         [(128, 4, "bf16", 128, False, True), (64, 12, "f32", 32, True, False),
                          (96, 1, "bf16", 96, False, True), (192, 3, "f32", 64, False, True),
                          (256, 2, "bf16", 256, True, True), (128, 8, "f32", 14, False, False),
                          (64, 33, "bf16", 0, False, True), (128, 1, "bf16", 0, False, False),
                          (96, 2, "f32", 10, True, True),
                          (96, 2, "bf16", 12, False, True), (192, 1, "f32", 190, False, False),
                          (256, 2, "bf16", 250, False, True)])
@pytest.mark.parametrize("kind", ["head", "position"])
@pytest.mark.parametrize("new", [None, [3, 0, 40, 1, 17, 0]])
def test_append(gpu, dim, kv, dtype, rot, interleaved, norm, kind, new):
    """values to the bit, keys to the rounding; every other row of the pool as it was; rows outside starts unread"""
    import torch
    lengths = [3, 25, 777, 64, 17, 0] if new else [3, 25, 777, 64, 17, 1]
    cache = Cache(lengths, kv, 24, dim, 30, kind, width=40)
    opt = _options(dim, 31, norm, rot, interleaved, 1.25)
    counts = new or [1] * 6
    first, behind = (2, 5) if new else (0, 0)
    total = first + sum(counts) + behind
    rows = rounded(O.fill_normal((total, 2 * kv, dim), 32, "kv"), dtype)
    rows[:first] = rows[total - behind:] = np.nan
    starts = first + np.concatenate([[0], np.cumsum(counts)])
    keys, values, table, lens = cache.device()
    before = [host_bits(keys.contiguous()).copy(), host_bits(values.contiguous()).copy()]
    t = _dev(rows, dtype)
    say("paged append", dict(dim=dim, kv=kv, dtype=dtype, rot=rot, kind=kind, new=new))
    gpu.paged_append(t[:, :kv], t[:, kv:], keys, values, table, lens, starts=dev_u32(starts) if new else None,
                     k_norm=None if opt["gamma"] is None else dev_f32(opt["gamma"]),
                     freqs=None if opt["freqs"] is None else dev_f32(opt["freqs"]), interleaved=interleaved,
                     amplitude=1.25)
    got_k, got_v = host(keys.contiguous()), host_bits(values.contiguous())
    bits_k = host_bits(keys.contiguous())
    written = np.zeros((cache.pages, 24), bool)
    for b, n in enumerate(counts):
        p = np.arange(lengths[b] - n, lengths[b])
        at = cache.table[b][p // 24], slice(None), p % 24
        written[at[0], at[2]] = True
        k, v = rows[starts[b]:starts[b + 1], :kv], rows[starts[b]:starts[b + 1], kv:]
        assert np.array_equal(got_v[at], O.pack_bf16(v).reshape(v.shape))
        base = normed(k, opt["gamma"])
        want = turn(base, p, opt["freqs"], interleaved, 1.25)
        size = pair_sizes(base, opt["freqs"], interleaved, 1.25)
        half = HALF_STEP["bf16"]
        tol = np.abs(want) * half * (1 + half) + (TURN_STEPS + NORM_STEPS) * U * size * (1 + half)
        assert (np.abs(got_k[at] - want) <= tol).all()
    keep = ~written[:, None, :, None]
    assert np.array_equal(np.where(keep, bits_k, 0), np.where(keep, before[0], 0))
    assert np.array_equal(np.where(keep, got_v, 0), np.where(keep, before[1], 0))


def test_append_tokens_without_a_place(gpu):
    """positions below zero, past the table or in no page of the pool are left out; the others are written"""
    import torch
    cache = Cache([10, 10, 10, 10, 10], 2, 4, 64, 33, width=3)
    keys, values, table, lens = cache.device()
    before = host_bits(values).copy()
    lens[0] = 2            # of three new tokens the first would be at -1
    lens[1] = 14           # 11 lies in the table's last page, 12 and 13 past it
    table[2, 2] = cache.pages
    table[3, 2] = -1
    lens[4] = -1
    v = rounded(O.fill_normal((15, 2, 64), 34, "v"), "bf16")
    starts = dev_u32(np.arange(0, 16, 3))
    say("paged append without a place")
    gpu.paged_append(_dev(v, "bf16"), _dev(v, "bf16"), keys, values, table, lens, starts=starts)
    got = host_bits(values)
    want = before.copy()
    bits = O.pack_bf16(v).reshape(v.shape)
    t = cache.table
    want[t[0, 0], :, 0], want[t[0, 0], :, 1] = bits[1], bits[2]
    want[t[1, 2], :, 3] = bits[3]
    want[t[2, 1], :, 3], want[t[3, 1], :, 3] = bits[6], bits[9]      # position 7; 8 and 9 have no page
    assert np.array_equal(got, want)


@pytest.mark.parametrize("starts", [[5, 3, 9, 2], [0, 100, 200, 300], [7, 7, 7, 7], [2 ** 31, 1, 0, 4]])
def test_append_odd_starts_stay_in_bounds(gpu, starts):
    """starts that decrease, pass the rows or are all one: rows are read and written in bounds only"""
    cache = Cache([12, 12, 12], 2, 4, 64, 35)
    keys, values, table, lens = cache.device()
    k = _dev(rounded(O.fill_normal((9, 2, 64), 36, "k"), "f32"), "f32")
    say("paged append odd starts", starts)
    gpu.paged_append(k, k, keys, values, table, lens, starts=dev_u32(np.array(starts, np.uint32)))
    assert np.isfinite(host(values)[cache.table[:, :3].ravel()]).all()


def test_serving_loop(gpu):
    """prompts appended in one call, then steps of append and decode for a padded batch, new pages handed out on
    the way; each step against float64 over what was appended, and against aigpu_decode_attention on a contiguous
    cache of the same rows. That one scores the newest key before its rounding, and a cached key of its fp32 angles
    may round to the neighbour: keys differ by a step of bf16, 2^-7 of themselves, at most, a score by scale
    sum |q| |k| 2^-7, and an average of values by twice the largest such change times the largest value"""
    import torch
    H, KV, D, page, steps = 8, 2, 128, 16, 20
    prompts = [37, 0, 5, 64, 150]
    opt = _options(D, 40, True, D)
    gk, gq = opt["gamma"], opt["gamma"]
    cache = Cache([n + steps if n else 0 for n in prompts], KV, page, D, 41, fill=False)
    cache.keys[:], cache.values[:] = np.nan, np.nan
    keys, values, table, lens = cache.device()
    rows = [(rounded(O.fill_normal((n + steps if n else 0, KV, D), 42, f"k{b}") if n else np.zeros((0, KV, D)), "bf16"),
             rounded(O.fill_normal((n + steps if n else 0, KV, D), 42, f"v{b}") if n else np.zeros((0, KV, D)), "bf16"))
            for b, n in enumerate(prompts)]
    lens.copy_(torch.tensor(prompts, dtype=torch.int32))
    starts = np.concatenate([[0], np.cumsum(prompts)])
    f, g = dev_f32(opt["freqs"]), dev_f32(gk)
    say("serving loop: prompts")
    gpu.paged_append(_dev(np.concatenate([r[0][:n] for r, n in zip(rows, prompts)]), "bf16"),
                     _dev(np.concatenate([r[1][:n] for r, n in zip(rows, prompts)]), "bf16"), keys, values, table,
                     lens, starts=dev_u32(starts), k_norm=g, freqs=f)
    cap = max(cache.lengths) + 1
    kc = torch.zeros((5, KV, cap, D), dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    live = [b for b, n in enumerate(prompts) if n]
    for b in live:      # the same prompts into the contiguous caches
        n = prompts[b]
        gpu.prefill(_dev(np.zeros((n, H, D), np.float32), "bf16"), _dev(rows[b][0][:n], "bf16"),
                    _dev(rows[b][1][:n], "bf16"), torch.zeros((n, H, D), device="cuda"), kc[b], vc[b], 0, H, KV, D,
                    q_norm=g, k_norm=g, freqs=f, rotary_dims=D)
    for step in range(steps):
        lens += (lens > 0).to(torch.int32)
        q = rounded(O.fill_normal((5, H, D), 43 + step, "q"), "bf16")
        new = [np.stack([rows[b][i][prompts[b] + step] if prompts[b] else np.zeros((KV, D), np.float32)
                         for b in range(5)]) for i in (0, 1)]
        out = torch.full((5, H, D), 7.0, device="cuda")
        say("serving loop: step", step)
        gpu.paged_append(_dev(new[0], "bf16"), _dev(new[1], "bf16"), keys, values, table, lens, k_norm=g, freqs=f)
        gpu.paged_decode(_dev(q, "bf16"), out, keys, values, table, lens, q_norm=g, freqs=f)
        got = host(out)
        assert (got[1] == 0).all()
        ref = torch.zeros((5, H, D), device="cuda")
        gpu.decode(_dev(q, "bf16"), _dev(new[0], "bf16"), _dev(new[1], "bf16"), ref, kc, vc,
                   dev_u32(np.array([n + step if n else 0 for n in prompts])), cap - 1, H, KV, D, q_norm=g, k_norm=g,
                   freqs=f, rotary_dims=D)
        ref = host(ref)
        hk, hv = host(keys), host(values)
        for b in live:
            n = prompts[b] + step + 1
            p = np.arange(n)
            at = cache.table[b][p // page], slice(None), p % page
            want, bound = decode64(q[b], hk[at].astype(np.float64), hv[at].astype(np.float64), n - 1, **opt)
            assert (np.abs(got[b] - want) <= bound).all()
            t = np.abs(turn(normed(q[b], gq)[None], [n - 1], opt["freqs"])[0]).reshape(KV, H // KV, D)
            change = np.einsum("kgd,pkd->kgp", t, np.abs(hk[at])).max(-1).reshape(H, 1) * D ** -0.5 * 2.0 ** -7
            assert (np.abs(got[b] - ref[b]) <= 2 * change * np.abs(hv[at]).max()).all()
            assert np.array_equal(hv[at], rows[b][1][:n])


def _graph_case(gpu, lengths, seed):
    import torch
    cache = Cache(lengths, 2, 16, 128, seed)
    opt = _options(128, seed, True, 128)
    q = rounded(O.fill_normal((len(lengths), 16, 128), seed, "q"), "bf16")
    return cache, opt, q, _dev(q, "bf16"), cache.device(), dev_f32(opt["gamma"]), dev_f32(opt["freqs"])


def test_captured_steps_follow_the_lengths(gpu):
    """append and decode in a graph with a workspace of its own, sized by the table: replayed as the lengths grow,
    with eager calls of other sizes between, every replay equal to the eager step to the bit"""
    import torch
    lengths = [4100, 17, 0, 900]
    cache, opt, q, dq, (keys, values, table, lens), g, f = _graph_case(gpu, lengths, 50)
    k = _dev(rounded(O.fill_normal((4, 2, 128), 51, "k"), "bf16"), "bf16")
    out = torch.zeros((4, 16, 128), device="cuda")
    room = gpu.paged_decode_workspace(dq, out, keys, values, table, lens)
    start = lens - 3 * (lens > 3).to(torch.int32)
    one = (lens > 0).to(torch.int32)

    def step(space):
        lens.add_(one)
        gpu.paged_append(k, k, keys, values, table, lens, k_norm=g, freqs=f)
        gpu.paged_decode(dq, out, keys, values, table, lens, q_norm=g, freqs=f, workspace=space)

    lens.copy_(start)
    want = []
    for _ in range(3):
        step(None)
        want.append(host(out).copy())
    lens.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(room)
    other = _graph_case(gpu, [7000, 31, 64], 52)
    for i in range(3):
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(out), want[i]), i
        _check_decode(_decode(gpu, other[0], other[2], "bf16", other[1]), other[0], other[2], other[1])


def test_two_graphs_with_a_workspace_each_replay_together(gpu):
    import torch
    made, graphs, streams = [], [], []
    for i, lengths in enumerate(([3000, 60], [2500, 2, 1800])):
        cache, opt, q, dq, dev, g, f = _graph_case(gpu, lengths, 60 + i)
        out = torch.zeros((len(lengths), 16, 128), device="cuda")
        gpu.paged_decode(dq, out, *dev, q_norm=g, freqs=f)
        want = host(out).copy()
        room = gpu.paged_decode_workspace(dq, out, *dev)
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            gpu.paged_decode(dq, out, *dev, q_norm=g, freqs=f, workspace=room, stream=side.cuda_stream)
        made.append((out, want, dq, dev, g, f, room))
        graphs.append(graph)
        streams.append(side)
    for _ in range(3):
        for m in made:
            m[0].fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(10):
            for graph, side in zip(graphs, streams):
                with torch.cuda.stream(side):
                    graph.replay()
        torch.cuda.synchronize()
        for m in made:
            assert np.array_equal(host(m[0]), m[1])


def test_calls_on_many_streams_at_once(gpu):
    import torch
    cases = [_graph_case(gpu, lengths, 70 + i) for i, lengths in enumerate(([5000, 300], [4000, 9, 2000]))]
    want = [_decode(gpu, c[0], c[2], "bf16", c[1]) for c in cases]
    # more streams than have a scratch of their own
    sides = [torch.cuda.Stream() for _ in range(12)]
    outs = [[torch.full((len(c[0].lengths), 16, 128), 7.0, device="cuda") for c in cases] for _ in sides]
    torch.cuda.synchronize()
    for _ in range(8):
        for side, row in zip(sides, outs):
            for c, out in zip(cases, row):
                gpu.paged_decode(c[3], out, *c[4], q_norm=c[5], freqs=c[6], stream=side.cuda_stream)
    torch.cuda.synchronize()
    for row in outs:
        for out, w in zip(row, want):
            assert np.array_equal(host(out), w)


def test_gpu_refusals(gpu):
    """what only GPU tensors get far enough to show; nothing is launched"""
    import torch
    cache = Cache([20, 5000], 2, 16, 128, 80)
    keys, values, table, lens = cache.device()
    q, out = torch.zeros((2, 16, 128), device="cuda"), torch.zeros((2, 16, 128), device="cuda")
    f, g = dev_f32(O.rotary_frequencies(128, 1e6)), torch.ones(128, device="cuda")
    kv = torch.zeros((2, 2, 128), device="cuda")

    def decode(q=q, out=out, keys=keys, values=values, table=table, lens=lens, **kw):
        return lambda: gpu.paged_decode(q, out, keys, values, table, lens, **kw)

    def append(k=kv, v=kv, keys=keys, values=values, table=table, lens=lens, **kw):
        return lambda: gpu.paged_append(k, v, keys, values, table, lens, **kw)

    odd = torch.zeros((4, 2, 16, 132), dtype=torch.bfloat16, device="cuda")[..., :128]
    off = torch.zeros(4 * 2 * 16 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 2, 16, 128)
    tiny = torch.zeros((4, 2, 16, 80), dtype=torch.bfloat16, device="cuda")
    bad = [decode(max_length=table.shape[1] * 16 + 1), decode(max_length=-1), decode(window=-1),
           decode(scale=float("inf")), decode(scale=-1.0), decode(amplitude=float("nan"), freqs=f),
           decode(q=q[:, :15], out=out[:, :15].contiguous()), decode(q=q[:1]), decode(q=q.half()),
           decode(out=out.bfloat16()), decode(out=out[:, :, :64]), decode(output_gate=True),
           decode(lens=lens.long()), decode(table=table.long()), decode(table=table.t()), decode(lens=lens[:1]),
           decode(keys=keys.float(), values=values.float()), decode(values=values[:-1]), decode(keys=odd, values=odd),
           decode(keys=off, values=off), decode(q=q[..., :80], out=out[..., :80].contiguous(), keys=tiny, values=tiny),
           decode(out=q), decode(q_norm=g[:64]), decode(q_norm=g.double()), decode(freqs=f, rotary_dims=63),
           decode(freqs=f, rotary_dims=130), decode(freqs=f[:10], rotary_dims=64),
           append(k=kv[:1], v=kv[:1]), append(k=kv[:, :1], v=kv[:, :1]), append(v=kv.bfloat16()),
           append(starts=lens), append(starts=torch.zeros(3, device="cuda")), append(k_norm=g[:64]),
           append(k=kv[:1].expand(2, 2, 128)), append(keys=off, values=off), append(freqs=f, amplitude=-1.0)]
    for i, call in enumerate(bad):
        with pytest.raises((gpu.AiGpuError, ValueError, TypeError)):
            call()
            pytest.fail(f"case {i} was taken")
    room = gpu.paged_decode_workspace(q, out, keys, values, table, lens)
    for space in (room[:-1], torch.cat([room, room])[8:]):
        with pytest.raises(gpu.AiGpuError):
            gpu.paged_decode(q, out, keys, values, table, lens, workspace=space)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.zero_()
        with pytest.raises(gpu.AiGpuError):      # the backend's scratch may move
            gpu.paged_decode(q, out, keys, values, table, lens)
    # nothing to do is no error
    gpu.paged_append(kv[:0], kv[:0], keys, values, table[:0], lens[:0])
    gpu.paged_decode(q[:0], out[:0], keys, values, table[:0], lens[:0])
