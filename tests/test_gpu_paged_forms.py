"""GPU tests of the forms that the rotary and paged entries take for other sizes
than test_gpu_paged.py's: appends of several tokens a workgroup and of more rows
than its lanes hold, both ways to join a decode's parts under graphs, streams
and threads, backward in bf16, and rows that lie between one another."""
import threading

import numpy as np
import pytest

from gpu_util import dev_f32, dev_u32, host, host_bits, say
from oracle import oracle as O
from paged_products import tight64
from paged_util import HALF_STEP, NORM_STEPS, TURN_STEPS, U, Cache, normed, pair_sizes, rounded, turn
from test_gpu_paged import _dev, _options
from test_gpu_rotary import _check as _check_rotary
from test_gpu_rotary import _run as _run_rotary

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("dim,kv,dtype,rot,interleaved,norm,counts,first,behind", [
    (64, 1, "bf16", 64, False, True, [1024], 0, 0),                       # two tokens a workgroup
    (64, 1, "bf16", 64, False, True, [700, 0, 401, 3, 432, 1], 0, 0),     # three, the last of 512.33 tiles cut short
    (64, 2, "f32", 32, True, False, [2000, 63, 1, 2050], 5, 9),           # eight
    (64, 1, "bf16", 64, False, True, [1] * 300 + [0] * 5 + [4000, 3957], 3, 2),  # sixteen, many sequences a tile
    (128, 1, "f32", 14, False, True, [5000, 0, 3200, 7], 0, 0),           # sixteen, an uneven rotation
    (96, 2, "bf16", 96, False, True, [900, 900], 1, 0),                   # three
    (192, 1, "bf16", 190, False, True, [1999], 0, 0),                     # three of four that the lanes hold
    (256, 4, "f32", 256, True, True, [1100], 0, 31),                      # two
    (128, 40, "bf16", 128, False, True, [30, 1, 70], 0, 2),               # 80 rows a token: a second trip of the lanes
    (128, 40, "f32", 128, False, False, [600, 501], 0, 0),
    (64, 65, "bf16", 0, False, False, [40], 0, 0),
    (256, 20, "bf16", 128, True, True, [9, 60], 0, 0),
    (96, 41, "f32", 10, False, True, [33, 0, 20], 4, 4),
    (192, 17, "bf16", 64, False, True, [25, 26], 0, 0),
])
@pytest.mark.parametrize("kind", ["head", "position"])
def test_append_of_many_rows(gpu, dim, kv, dtype, rot, interleaved, norm, counts, first, behind, kind):
    """values to the bit, keys to the rounding; every other row of the pool as it was; rows outside starts unread"""
    import torch
    lengths = [n + (37 * b) % 90 for b, n in enumerate(counts)]
    cache = Cache(lengths, kv, 24, dim, 130, kind, fill=False)
    opt = _options(dim, 131, norm, rot, interleaved, 1.25)
    starts = first + np.concatenate([[0], np.cumsum(counts)])
    total = int(starts[-1]) + behind
    rows = rounded(O.fill_normal((total, 2 * kv, dim), 132, "kv"), dtype)
    rows[:first] = rows[total - behind:] = np.nan
    cache.keys[:] = cache.values[:] = 0.5
    keys, values, table, lens = cache.device()
    t = _dev(rows, dtype)
    say("paged append", dict(dim=dim, kv=kv, dtype=dtype, rot=rot, kind=kind, counts=counts[:6]))
    gpu.paged_append(t[:, :kv], t[:, kv:], keys, values, table, lens, starts=dev_u32(starts),
                     k_norm=None if opt["gamma"] is None else dev_f32(opt["gamma"]),
                     freqs=None if opt["freqs"] is None else dev_f32(opt["freqs"]), interleaved=interleaved,
                     amplitude=1.25)
    got_k, got_v = host(keys.contiguous()), host_bits(values.contiguous())
    written = np.zeros((cache.pages, 24), bool)
    half = HALF_STEP["bf16"]
    for b, n in enumerate(counts):
        p = np.arange(lengths[b] - n, lengths[b])
        at = cache.table[b][p // 24], slice(None), p % 24
        assert not written[at[0], at[2]].any()
        written[at[0], at[2]] = True
        k, v = rows[starts[b]:starts[b + 1], :kv], rows[starts[b]:starts[b + 1], kv:]
        assert np.array_equal(got_v[at], O.pack_bf16(v).reshape(v.shape)), b
        base = normed(k, opt["gamma"])
        want = turn(base, p, opt["freqs"], interleaved, 1.25)
        tol = np.abs(want) * half * (1 + half) + \
            (TURN_STEPS + NORM_STEPS) * U * pair_sizes(base, opt["freqs"], interleaved, 1.25) * (1 + half)
        assert (np.abs(got_k[at] - want) <= tol).all(), b
    same = np.broadcast_to(~written[:, None, :, None], got_k.shape)
    assert (got_k[same] == 0.5).all() and (got_v[same] == 0x3F00).all()


# ------------------------------------------------------------------- decode, joined either way
JOINS = {"in the launch": (8, 4, 1), "by a second launch": (16, 2, 2)}   # heads, kv heads, launches of a decode


def _case(gpu, lengths, seed, join):
    """inputs whose decodes leave parts in several workgroups, and the call"""
    import torch
    heads, kv, launches = JOINS[join]
    cache = Cache(lengths, kv, 16, 128, seed)
    opt = _options(128, seed, True, 128)
    q = rounded(O.fill_normal((len(lengths), heads, 128), seed, "q"), "bf16")
    dq, device, g, f = _dev(q, "bf16"), cache.device(), dev_f32(opt["gamma"]), dev_f32(opt["freqs"])
    out = torch.zeros((len(lengths), heads, 128), device="cuda")

    def call(to=out, **kw):
        gpu.paged_decode(dq, to, *device, q_norm=g, freqs=f, **kw)

    say("paged decode joined", join, lengths)
    before = gpu.counters()["launches"]
    call()
    assert gpu.counters()["launches"] - before == launches
    want = host(out).copy()
    for b, n in enumerate(lengths):
        if n:
            exact, bound = tight64(q[b].astype(np.float64), *cache.rows(b), n - 1, **opt)
            assert (np.abs(want[b] - exact) <= bound).all(), b
    room = gpu.paged_decode_workspace(dq, out, *device)
    return dict(call=call, out=out, want=want, room=room, device=device, cache=cache, kv=kv, g=g, f=f)


@pytest.mark.parametrize("join", JOINS)
def test_captured_steps_of_either_join(gpu, join):
    """append and decode replayed as the lengths grow, eager decodes of other sizes between the replays; every replay
    equal to the eager step to the bit"""
    import torch
    c = _case(gpu, [4100, 17, 0, 900], 150, join)
    keys, values, table, lens = c["device"]
    k = _dev(rounded(O.fill_normal((4, c["kv"], 128), 151, "k"), "bf16"), "bf16")
    start, one = lens - 3 * (lens > 3).to(torch.int32), (lens > 0).to(torch.int32)

    def step(**kw):
        lens.add_(one)
        gpu.paged_append(k, k, keys, values, table, lens, k_norm=c["g"], freqs=c["f"])
        c["call"](**kw)

    lens.copy_(start)
    want = []
    for _ in range(3):
        step()
        want.append(host(c["out"]).copy())
    lens.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(workspace=c["room"])
    other = _case(gpu, [7000, 31, 64], 152, join)
    for i in range(3):
        c["out"].fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(c["out"]), want[i]), i
        other["call"]()
        assert np.array_equal(host(other["out"]), other["want"])


@pytest.mark.parametrize("join", JOINS)
def test_two_graphs_of_either_join_replay_together(gpu, join):
    import torch
    made = []
    for i, lengths in enumerate(([3000, 60], [2500, 2, 1800])):
        c = _case(gpu, lengths, 160 + i, join)
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            c["call"](workspace=c["room"], stream=side.cuda_stream)
        made.append((c, graph, side))
    for _ in range(3):
        for c, _, _ in made:
            c["out"].fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(10):
            for _, graph, side in made:
                with torch.cuda.stream(side):
                    graph.replay()
        torch.cuda.synchronize()
        for c, _, _ in made:
            assert np.array_equal(host(c["out"]), c["want"])


@pytest.mark.parametrize("join", JOINS)
def test_many_streams_of_either_join(gpu, join):
    """more streams than have a scratch of their own"""
    import torch
    cases = [_case(gpu, lengths, 170 + i, join) for i, lengths in enumerate(([5000, 300], [4000, 9, 2000]))]
    sides = [torch.cuda.Stream() for _ in range(12)]
    outs = [[torch.full_like(c["out"], 7.0) for c in cases] for _ in sides]
    torch.cuda.synchronize()
    for _ in range(8):
        for side, row in zip(sides, outs):
            for c, out in zip(cases, row):
                c["call"](out, stream=side.cuda_stream)
    torch.cuda.synchronize()
    for row in outs:
        for out, c in zip(row, cases):
            assert np.array_equal(host(out), c["want"])


@pytest.mark.parametrize("join", JOINS)
def test_threads_on_their_per_thread_streams(gpu, join):
    """one handle, a stream in each thread that goes with it, one scratch between them"""
    import torch
    per_thread = 2
    cases = [_case(gpu, lengths, 180 + i, join) for i, lengths in enumerate(([5000, 300], [4000, 9, 2000]))]
    outs = [[torch.full_like(c["out"], 7.0) for _ in range(100)] for c in cases]
    torch.cuda.synchronize()
    failures = []

    def work(c, row):
        try:
            for out in row:
                c["call"](out, stream=per_thread)
        except Exception as e:
            failures.append(e)

    for at in range(0, 100, 10):     # threads that end with their last call's work just queued
        threads = [threading.Thread(target=work, args=(c, row[at:at + 10])) for c, row in zip(cases, outs)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    torch.cuda.synchronize()
    assert not failures
    for c, row in zip(cases, outs):
        for out in row:
            assert np.array_equal(host(out), c["want"])


@pytest.mark.parametrize("join", JOINS)
def test_a_growing_conversation_keeps_its_scratch(gpu, join):
    """max_length follows the length, as a serving loop gives it: after the first call nothing is allocated"""
    import torch
    heads, kv, _ = JOINS[join]
    cache = Cache([6000], kv, 16, 128, 190)
    keys, values, table, lens = cache.device()
    q = rounded(O.fill_normal((1, heads, 128), 191, "q"), "f32")
    dq, out = dev_f32(q), torch.zeros((1, heads, 128), device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    held = None
    for n in list(range(1, 200)) + list(range(200, 6001, 40)) + [6000]:
        with torch.cuda.stream(side):
            lens.fill_(n)
            gpu.paged_decode(dq, out, keys, values, table, lens, max_length=n)
        held = held or gpu.lib().aigpu_allocated_bytes()
        assert gpu.lib().aigpu_allocated_bytes() == held
        if n in (1, 33, 199, 3000, 6000):
            side.synchronize()
            k, v = cache.rows(0, n)
            want, bound = tight64(q[0].astype(np.float64), k, v, n - 1)
            assert (np.abs(host(out)[0] - want) <= bound).all(), n


def test_gated_views_narrower_than_their_gates(gpu):
    """refused: their gates lie outside them, the last one's past the buffer"""
    import torch
    cache = Cache([20, 50, 3], 2, 16, 128, 195)
    out = torch.zeros((3, 4, 128), device="cuda")
    wide = torch.zeros((3, 4, 256), device="cuda")
    for q in (wide[..., :128], wide[..., 128:], torch.zeros((3, 8, 128), device="cuda")[:, 1::2]):
        with pytest.raises(ValueError):
            gpu.paged_decode(q, out, *cache.device(), output_gate=True)


# ------------------------------------------------------------------- rotary
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 32, 128, 128), (37, 5, 64, 32), (300, 40, 192, 64), (9, 3, 17, 6)])
def test_backward_in_bf16(gpu, interleaved, tokens, heads, dim, rot):
    dy = rounded(O.fill_normal((tokens, heads, dim), rot, "dy"), "bf16")
    freqs = O.rotary_frequencies(rot, 1e6)
    positions = np.random.default_rng(dim).integers(0, 200000, tokens).astype(np.uint32)
    got = _run_rotary(gpu, dy, positions, freqs, "bf16", interleaved=interleaved, amplitude=1.25, backward=True)
    _check_rotary(got, dy, positions, freqs, interleaved, 1.25, "bf16", sign=-1.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads", [(1, 6), (211, 6), (211, 1)])
def test_one_half_of_wider_heads_into_the_other(gpu, dtype, interleaved, tokens, heads):
    dim, freqs = 64, O.rotary_frequencies(48, 1e4)
    x = rounded(O.fill_normal((tokens, heads, 2 * dim), 8, "x"), dtype)
    positions = np.arange(100, 100 + tokens, dtype=np.uint32)
    for a, b in ((slice(None, dim), slice(dim, None)), (slice(dim, None), slice(None, dim))):
        wide = _dev(x, dtype)
        say("rotary of a half", tokens, heads, dtype, interleaved)
        gpu.rotary(wide[..., a], wide[..., b], dev_f32(freqs), positions=dev_u32(positions), interleaved=interleaved)
        got = host(wide)
        assert np.array_equal(got[..., a], x[..., a])
        _check_rotary(got[..., b], x[..., a], positions, freqs, interleaved, 1.0, dtype)
