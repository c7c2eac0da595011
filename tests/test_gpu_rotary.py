"""GPU parity of aigpu_rotary against float64: both pair layouts, part of the
head, strides and alignments of either tensor, in place, far positions,
backward, and its refusals."""
import numpy as np
import pytest

from common import gammas
from gpu_util import dev_f32, dev_u32, host, say
from oracle import oracle as O
from paged_util import HALF_STEP, TURN_STEPS, U, pair_sizes, rounded, turn

pytestmark = pytest.mark.gpu


def _dtype(name):
    import torch
    return torch.bfloat16 if name == "bf16" else torch.float32


def _check(got, x, positions, freqs, interleaved, amplitude, dtype, sign=1.0):
    want = turn(x, positions, freqs, interleaved, amplitude, sign)
    tol = np.abs(want) * HALF_STEP[dtype] * (1 + HALF_STEP[dtype]) + \
        TURN_STEPS * U * pair_sizes(x, freqs, interleaved, amplitude)
    rot = 2 * len(freqs)
    assert np.array_equal(got[..., rot:], np.asarray(x, np.float32)[..., rot:])
    err = np.abs(got - want)
    assert (err <= tol).all(), (err - tol).max()


def _run(gpu, x, positions, freqs, dtype, **kw):
    import torch
    t = torch.from_numpy(x).cuda().to(_dtype(dtype))
    out = torch.full_like(t, float("nan"))
    say("rotary", x.shape, len(freqs), dtype, kw)
    gpu.rotary(t, out, dev_f32(freqs), positions=None if positions is None else dev_u32(positions), **kw)
    return host(out)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 128), (64, 32), (96, 96), (192, 64), (256, 256), (80, 24), (17, 6), (2, 2),
                                     (128, 14), (640, 640)])
def test_shapes(gpu, dtype, interleaved, dim, rot):
    for tokens, heads in ((1, 1), (1, 32), (37, 5), (200, 40)):
        x = rounded(O.fill_normal((tokens, heads, dim), dim + rot, "x"), dtype)
        freqs = O.rotary_frequencies(rot, 1e6)
        positions = np.random.default_rng(tokens).integers(0, 200000, tokens).astype(np.uint32)
        got = _run(gpu, x, positions, freqs, dtype, interleaved=interleaved, amplitude=1.25)
        _check(got, x, positions, freqs, interleaved, 1.25, dtype)


def test_many_tokens_and_heads(gpu):
    for tokens, heads, dim in ((3001, 8, 128), (5, 1001, 64), (70000, 1, 64)):
        x = rounded(O.fill_normal((tokens, heads, dim), 3, "x"), "bf16")
        freqs = O.rotary_frequencies(dim, 1e4)
        _check(_run(gpu, x, None, freqs, "bf16", start=17), x, 17 + np.arange(tokens), freqs, False, 1.0, "bf16")


def test_more_tiles_than_one_side_of_a_grid(gpu):
    """2^24 + 7 tokens that take a tile each: 2^32 threads and more, 17 GB of output over rows of x one element apart"""
    import torch
    n, heads, dim, freqs = 2 ** 24 + 7, 2, 257, np.ones(1, np.float32)
    x = O.fill_normal((n + heads * dim,), 6, "x")
    flat = torch.from_numpy(x).cuda()
    out = torch.empty((n, heads, dim), dtype=torch.bfloat16, device="cuda")
    picked = np.array([0, 1, 2 ** 23 - 1, 2 ** 23, 2 ** 23 + 1, 2 ** 24 - 1, 2 ** 24, 2 ** 24 + 6])
    out[picked] = float("nan")
    say("rotary", n, heads, dim)
    gpu.rotary(flat.bfloat16().as_strided((n, heads, dim), (1, dim, 1)), out, dev_f32(freqs), start=5)
    rows = rounded(x, "bf16")[picked[:, None] + np.arange(heads * dim)].reshape(len(picked), heads, dim)
    _check(host(out[torch.from_numpy(picked).cuda()]), rows, 5 + picked, freqs, False, 1.0, "bf16")


@pytest.mark.parametrize("position", [0, 1, 131071, 2 ** 24 + 1, 2 ** 31, 2 ** 32 - 1])
def test_far_positions(gpu, position):
    """float64 holds the angle of position 2^32 to 2^-53 2^32 radians, within TURN_STEPS"""
    x = rounded(O.fill_normal((1, 3, 128), 5, "x"), "f32")
    freqs = O.rotary_frequencies(128, 1e6)
    _check(_run(gpu, x, np.array([position], np.uint32), freqs, "f32"), x, [position], freqs, False, 1.0, "f32")
    _check(_run(gpu, x, None, freqs, "f32", start=position), x, [position], freqs, False, 1.0, "f32")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_alignment_and_in_place(gpu, dtype, interleaved):
    """heads inside wider rows, a head-major tensor, rows off 16 bytes, in place; elements outside stay"""
    import torch
    tokens, heads, dim, rot = 9, 6, 64, 48
    freqs = O.rotary_frequencies(rot, 1e4)
    positions = np.arange(100, 100 + tokens, dtype=np.uint32)
    x = rounded(O.fill_normal((tokens, heads, dim), 8, "x"), dtype)
    f, p = dev_f32(freqs), dev_u32(positions)

    def place(kind):
        """a view of that shape and the buffer round it"""
        t = _dtype(dtype)
        if kind == "dense":
            buf = torch.full((tokens, heads, dim), 7.0, dtype=t, device="cuda")
            return buf, buf
        if kind == "wide":
            buf = torch.full((tokens, 3 * heads, dim), 7.0, dtype=t, device="cuda")
            return buf[:, heads:2 * heads], buf
        if kind == "gate":      # each head's row followed by another half
            buf = torch.full((tokens, heads, 2 * dim), 7.0, dtype=t, device="cuda")
            return buf[..., :dim], buf
        if kind == "head-major":
            buf = torch.full((heads, tokens, dim), 7.0, dtype=t, device="cuda")
            return buf.transpose(0, 1), buf
        buf = torch.full((tokens * heads * (dim + 1) + 1,), 7.0, dtype=t, device="cuda")
        return buf[1:].view(tokens, heads, dim + 1)[..., :dim], buf    # odd

    kinds = ["dense", "wide", "gate", "head-major", "odd"]
    for a in kinds:
        for b in kinds:
            src, _ = place(a)
            dst, whole = place(b)
            src.copy_(torch.from_numpy(x))
            say("rotary strides", a, b)
            gpu.rotary(src, dst, f, positions=p, interleaved=interleaved)
            _check(host(dst.contiguous()), x, positions, freqs, interleaved, 1.0, dtype)
            dst.fill_(7.0)
            assert bool((whole == 7.0).all())
        src, whole = place(a)
        src.copy_(torch.from_numpy(x))
        gpu.rotary(src, src, f, positions=p, interleaved=interleaved)
        _check(host(src.contiguous()), x, positions, freqs, interleaved, 1.0, dtype)
        src.fill_(7.0)
        assert bool((whole == 7.0).all())
    # side by side in the same rows
    buf = torch.zeros((tokens, 2 * heads, dim), dtype=_dtype(dtype), device="cuda")
    buf[:, heads:] = torch.from_numpy(x).cuda()
    gpu.rotary(buf[:, heads:], buf[:, :heads], f, positions=p, interleaved=interleaved)
    _check(host(buf[:, :heads].contiguous()), x, positions, freqs, interleaved, 1.0, dtype)
    assert np.array_equal(host(buf[:, heads:].contiguous()), x)


@pytest.mark.parametrize("interleaved", [False, True])
def test_backward(gpu, interleaved):
    """against the formula, and against differences of the forward: it is linear, so a unit step has no error of
    second order, and <dy, R e_i> = (R^T dy)_i up to the roundings of both sides"""
    tokens, heads, dim, rot, A = 3, 2, 32, 20, 1.2
    freqs = O.rotary_frequencies(rot, 1e4)
    positions = np.array([0, 77, 90001], np.uint32)
    dy = rounded(O.fill_normal((tokens, heads, dim), 9, "dy"), "f32")
    got = _run(gpu, dy, positions, freqs, "f32", interleaved=interleaved, amplitude=A, backward=True)
    _check(got, dy, positions, freqs, interleaved, A, "f32", sign=-1.0)
    x = rounded(O.fill_normal((tokens, heads, dim), 9, "x"), "f32")
    y0 = _run(gpu, x, positions, freqs, "f32", interleaved=interleaved, amplitude=A).astype(np.float64)
    for i in range(dim):
        e = x.copy()
        e[..., i] += 1.0
        step = (e - x)[..., i].astype(np.float64)   # exact by construction of both
        y1 = _run(gpu, e, positions, freqs, "f32", interleaved=interleaved, amplitude=A).astype(np.float64)
        slope = ((y1 - y0) * dy).sum(-1) / step
        # y1 and y0 round by TURN_STEPS of their pairs each (|x| + 1 bounds a pair's half)
        tol = (2 * (TURN_STEPS + 1) * U * 2 * A * (np.abs(x).max() + 1) * np.abs(dy).sum(-1) / step
               + 2 * TURN_STEPS * U * A * np.abs(dy).sum(-1))
        assert (np.abs(slope - got[..., i]) <= tol).all()


def test_attention_over_rotated_rows(gpu):
    """rotary of q and keys, then aigpu_attention_device over them: the chain
    that the fused entries run in one, here with interleaved pairs"""
    import torch
    T, H, KV, D = 65, 4, 2, 64
    freqs, _ = gpu.rotary_frequencies(D, 1e4, "linear", factor=2.0)
    q, k = (rounded(O.fill_normal((T, h, D), 10, n), "f32") for h, n in ((H, "q"), (KV, "k")))
    v = O.fill_normal((T, KV, D), 10, "v")
    dq, dk, f = dev_f32(q), dev_f32(k), dev_f32(freqs)
    gpu.rotary(dq, dq, f, interleaved=True)
    gpu.rotary(dk, dk, f, interleaved=True)
    out = torch.zeros((T, H, D), device="cuda")
    gpu.attention_device(dq, dk, dev_f32(v), out, T, 0, H, KV, D, D, KV * D, D)
    from common import assert_f32_parity, attention_fp64
    at = np.arange(T)
    ref = attention_fp64(turn(q, at, freqs, True).reshape(-1), turn(k, at, freqs, True), v, T, 0, H, KV, D, D, 0)
    assert_f32_parity(ref, host(out), "rotated attention")


def test_same_inputs_same_bits_and_streams(gpu):
    import torch
    x = torch.randn((501, 32, 128), device="cuda").to(torch.bfloat16)
    f = dev_f32(O.rotary_frequencies(128, 1e6))
    a, b = torch.empty_like(x), torch.empty_like(x)
    gpu.rotary(x, a, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gpu.rotary(x, b, f)
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    c = torch.zeros_like(x)
    with torch.cuda.graph(graph):
        gpu.rotary(x, c, f)
    for _ in range(3):
        c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, c)
        gpu.rotary(x, b, f, backward=True)


def test_empty(gpu):
    import torch
    f = dev_f32(O.rotary_frequencies(64, 1e6))
    for shape in ((0, 4, 64), (4, 0, 64)):
        x = torch.zeros(shape, device="cuda")
        gpu.rotary(x, x, f)


def test_gpu_refusals(gpu):
    """what only a GPU tensor gets far enough to show; nothing is launched"""
    import torch
    x = torch.zeros((4, 2, 64), device="cuda")
    f = dev_f32(O.rotary_frequencies(64, 1e6))
    flat = torch.zeros(4 * 2 * 64 + 64, device="cuda")
    a = flat[:512].view(4, 2, 64)
    bad = [lambda: gpu.rotary(a, flat[64:576].view(4, 2, 64), f),                  # overlaps
           lambda: gpu.rotary(x, x[:, :1].expand(4, 2, 64), f),                    # broadcast out
           lambda: gpu.rotary(x[:, :1].expand(4, 2, 64), x, f),
           lambda: gpu.rotary(x, x, f, rotary_dims=63),
           lambda: gpu.rotary(x, x, f, rotary_dims=66),
           lambda: gpu.rotary(x, x, f, rotary_dims=0),
           lambda: gpu.rotary(x, x, f, amplitude=float("nan")),
           lambda: gpu.rotary(x, x, f, amplitude=-1.0),
           lambda: gpu.rotary(x, x, f, start=2 ** 32 - 2),
           lambda: gpu.rotary(x, x, f, start=-1),
           lambda: gpu.rotary(x, x, f, positions=torch.zeros(4, dtype=torch.int64, device="cuda")),
           lambda: gpu.rotary(x, x, f, positions=torch.zeros(3, dtype=torch.int32, device="cuda")),
           lambda: gpu.rotary(x.half(), x.half(), f),
           lambda: gpu.rotary(x, torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda"), f),
           lambda: gpu.rotary(x, x, f.double()),
           lambda: gpu.rotary(x.transpose(1, 2), x.transpose(1, 2), f)]
    for i, call in enumerate(bad):
        with pytest.raises((gpu.AiGpuError, ValueError, TypeError)):
            call()
            pytest.fail(f"case {i} was taken")
