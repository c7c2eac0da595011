"""Attention of packed documents on the GPU, against float64."""
import numpy as np
import pytest

from gpu_util import dev_bf16, dev_f32, host, say
from oracle import oracle as O
from packed_util import document64
from paged_util import rounded

pytestmark = pytest.mark.gpu
TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"), ("f32", "bf16")]


def dev(x, dtype):
    return dev_bf16(O.pack_bf16(x)) if dtype == "bf16" else dev_f32(x)


def vector(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts_of(counts, first=0):
    return np.concatenate([[first], first + np.cumsum(counts)]).astype(np.int64).tolist()


def run(gpu, new, heads, kv, dim, dtype="bf16", out="bf16", past=None, prefix=None, window=0, cap=0.0, biased=False,
        first=0, behind=0, seed=1, size=1.0, workspace=False):
    """one call over documents of `new` tokens behind `past` keys each, checked; returns the call's output"""
    import torch
    lengths = [n + p for n, p in zip(new, past or [0] * len(new))]
    q = rounded(size * O.fill_normal((first + sum(new) + behind, heads, dim), seed, "q"), dtype)
    rows = first + sum(lengths) + behind
    k, v = (rounded(O.fill_normal((rows, kv, dim), seed, x), dtype) for x in "kv")
    # rows of no document hold what must not be read
    for x in (q, k, v):
        x[:first], x[len(x) - behind:] = np.nan, np.nan
    starts, key_starts = starts_of(new, first), starts_of(lengths, first)
    slopes = (2.0 ** -np.linspace(0.5, 7, heads)).astype(np.float32) if biased else None
    res = torch.full((len(q), heads, dim), 3.0, device="cuda", dtype=torch.bfloat16 if out == "bf16" else torch.float32)
    tensors = dev(q, dtype), dev(k, dtype), dev(v, dtype), res
    how = dict(starts=vector(starts), key_starts=vector(key_starts) if past else None)
    say("packed", new, heads, kv, dim, dtype, out, past, prefix, window, cap, biased)
    work = gpu.packed_attention_workspace(*tensors, **how) if workspace else None
    gpu.packed_attention(*tensors, **how, prefix=None if prefix is None else vector(prefix), window=window, cap=cap,
                         slopes=None if slopes is None else dev_f32(slopes), workspace=work)
    got = host(res)
    assert (got[:first] == 3).all() and (got[len(got) - behind:] == 3).all()
    for b, n in enumerate(new):
        at, ka = starts[b], key_starts[b]
        want, bound = document64(q[at:at + n], k[ka:ka + lengths[b]], v[ka:ka + lengths[b]], dtype, out,
                                 prefix[b] if prefix else 0, window, cap, slopes)
        far = np.abs(got[at:at + n] - want)
        assert (far <= bound).all(), (b, n, far.max(), np.nanmax(far / np.maximum(bound, 1e-300)), np.isnan(far).sum())
    return got


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype,out", TYPES)
def test_documents_of_many_lengths(gpu, dim, dtype, out):
    run(gpu, [1, 0, 5, 31, 32, 33, 64, 65, 130], 4, 2, dim, dtype, out, first=3, behind=2)


@pytest.mark.parametrize("heads,kv", [(12, 12), (8, 2), (16, 1), (24, 1), (5, 5), (6, 2), (40, 1)])
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f32", "f32")])
def test_heads_of_a_group(gpu, heads, kv, dtype, out):
    run(gpu, [3, 70, 17], heads, kv, 64, dtype, out)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("how", [dict(cap=2.0), dict(cap=50.0), dict(biased=True), dict(window=20), dict(window=1),
                                 dict(prefix=[40, 0, 90, 7]), dict(prefix=[1, 5, 64, 1000], window=33),
                                 dict(cap=5.0, biased=True, window=50, prefix=[0, 3, 100, 64])],
                         ids=lambda h: "-".join(h))
def test_forms(gpu, dim, dtype, out, how):
    run(gpu, [100, 7, 150, 64], 4, 2, dim, dtype, out, **how)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("how", [dict(), dict(window=100, biased=True), dict(cap=3.0, prefix=[10, 600, 0, 33])],
                         ids=lambda h: "-".join(h) or "plain")
def test_chunks_behind_their_keys(gpu, dim, dtype, out, how):
    """tokens that are the last of longer documents: few rows, whose keys are split"""
    run(gpu, [1, 9, 40, 3], 4, 2, dim, dtype, out, past=[700, 0, 1300, 64], **how)


def test_a_chunk_of_a_given_workspace(gpu):
    a = run(gpu, [1, 9], 4, 2, 64, "bf16", "f32", past=[3000, 5000])
    b = run(gpu, [1, 9], 4, 2, 64, "bf16", "f32", past=[3000, 5000], workspace=True)
    np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
def test_more_tokens_than_keys(gpu, dtype, out):
    """the first tokens stand before every key: zeros, or the prefix"""
    import torch
    H, D, n, m = 4, 64, 50, 20
    q, k, v = (rounded(O.fill_normal((x, h, D), 3, s), dtype) for x, h, s in ((n, H, "q"), (m, 2, "k"), (m, 2, "v")))
    say("packed more tokens", dtype, out)
    for prefix in (None, [6]):
        res = torch.full((n, H, D), 3.0, device="cuda", dtype=torch.bfloat16 if out == "bf16" else torch.float32)
        gpu.packed_attention(dev(q, dtype), dev(k, dtype), dev(v, dtype), res, starts=vector([0, n]),
                             key_starts=vector([0, m]), prefix=None if prefix is None else vector(prefix))
        got = host(res)
        want, bound = document64(q, k, v, dtype, out, prefix[0] if prefix else 0)
        assert (np.abs(got - want) <= bound).all()
        if prefix is None:
            assert (got[:n - m] == 0).all() and (got[n - m:] != 0).any()


def test_one_document_without_starts(gpu):
    import torch
    q, k, v = (rounded(O.fill_normal((x, h, 128), 4, s), "bf16") for x, h, s in ((33, 8, "q"), (90, 2, "k"), (90, 2, "v")))
    res = torch.empty((33, 8, 128), device="cuda", dtype=torch.bfloat16)
    say("packed without starts")
    gpu.packed_attention(dev(q, "bf16"), dev(k, "bf16"), dev(v, "bf16"), res)
    want, bound = document64(q, k, v, "bf16", "bf16")
    assert (np.abs(host(res) - want) <= bound).all()


def test_documents_without_keys_and_keys_without_tokens(gpu):
    import torch
    D = 64
    q, k, v = (rounded(O.fill_normal((x, 2, D), 5, s), "f32") for x, s in ((12, "q"), (30, "k"), (30, "v")))
    res = torch.full((12, 2, D), 3.0, device="cuda")
    say("packed empty sides")
    gpu.packed_attention(dev_f32(q), dev_f32(k), dev_f32(v), res, starts=vector([0, 5, 5, 12]),
                         key_starts=vector([0, 0, 10, 30]))
    got = host(res)
    assert (got[:5] == 0).all()
    want, bound = document64(q[5:], k[10:], v[10:], "f32", "f32")
    assert (np.abs(got[5:] - want) <= bound).all()


def test_starts_that_cannot_be_leave_out_alone(gpu):
    """starts that decrease or end past the tensors: such a document has no tokens, or no keys"""
    import torch
    x = dev_f32(O.fill_normal((20, 2, 64), 6, "x"))
    say("packed bad starts")
    res = torch.full((20, 2, 64), 3.0, device="cuda")
    gpu.packed_attention(x, x, x, res, starts=vector([0, 8, 40]))
    assert (host(res)[8:] == 3).all() and (host(res)[:8] != 3).any()
    res = torch.full((20, 2, 64), 3.0, device="cuda")
    gpu.packed_attention(x, x, x, res, starts=vector([0, 8, 20]), key_starts=vector([0, 8, 40]))
    assert (host(res)[8:] == 0).all()


def test_slices_of_one_products_rows(gpu):
    """q, k, v and out as slices of the same wider rows; head-major tensors give the same bits"""
    import torch
    H, KV, D, n = 4, 2, 128, 77
    rows = torch.randn((n, 2 * H + 2 * KV, D), device="cuda", dtype=torch.bfloat16)
    q, k, v, out = rows[:, :H], rows[:, H:H + KV], rows[:, H + KV:H + 2 * KV], rows[:, H + 2 * KV:]
    say("packed slices")
    gpu.packed_attention(q, k, v, out, starts=vector([0, 30, n]))
    dense = torch.empty((n, H, D), device="cuda", dtype=torch.bfloat16)
    gpu.packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), dense, starts=vector([0, 30, n]))
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    turned = torch.empty((H, n, D), device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    gpu.packed_attention(*major, turned, starts=vector([0, 30, n]))
    odd = torch.empty((n, H, D + 1), device="cuda", dtype=torch.bfloat16)[:, :, 1:]
    gpu.packed_attention(q, k, v, odd, starts=vector([0, 30, n]))
    torch.cuda.synchronize()
    assert torch.equal(out, dense) and torch.equal(turned, dense) and torch.equal(odd, dense)


def test_many_documents(gpu):
    """more documents than a wave looks at in one round"""
    r = np.random.default_rng(7)
    run(gpu, r.integers(0, 9, 300).tolist(), 2, 1, 64, "bf16", "f32")


def test_scores_of_any_size(gpu):
    """maxima that rise late, and scores far past the cap"""
    run(gpu, [300], 2, 2, 64, "f32", "f32", size=30.0)
    run(gpu, [300], 2, 2, 64, "f32", "f32", size=1e4, cap=10.0)


def test_captured(gpu):
    """captured once with and once without split keys, replayed over new inputs between eager calls"""
    import torch
    for new, past in (([40, 100], None), ([3, 5], [2000, 900])):
        lengths = [n + p for n, p in zip(new, past or [0, 0])]
        q, out = torch.randn((sum(new), 8, 128), device="cuda", dtype=torch.bfloat16), None
        k, v = (torch.randn((sum(lengths), 2, 128), device="cuda", dtype=torch.bfloat16) for _ in "kv")
        out = torch.empty((sum(new), 8, 128), device="cuda")
        how = dict(starts=vector(starts_of(new)), key_starts=vector(starts_of(lengths)) if past else None)
        work = gpu.packed_attention_workspace(q, k, v, out, **how)
        assert (work.numel() > 0) == bool(past) or not past
        say("packed captured", new, past)

        def step():
            gpu.packed_attention(q, k, v, out, **how, workspace=work if work.numel() else None, cap=30.0)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for _ in range(3):
            for t in (q, k, v):
                t.normal_()
            graph.replay()
            again = torch.empty_like(out)
            gpu.packed_attention(q, k, v, again, **how, cap=30.0)
            torch.cuda.synchronize()
            assert torch.equal(out, again)


def test_a_conversation(gpu):
    """prompt, append in 4 bits, a chunk over what the cache holds, a decode: used together"""
    import torch
    H, KV, D, cap = 8, 2, 128, 30.0
    prompts, chunk = [37, 90, 1], [5, 1, 16]
    total = [p + n for p, n in zip(prompts, chunk)]
    pages = 40
    pools = []
    for _ in "kv":
        pools += [torch.zeros((pages, KV, 16, D // 2), dtype=torch.uint8, device="cuda"),
                  torch.zeros((pages, KV, 16, D // 32), dtype=torch.float16, device="cuda")]
    table = torch.arange(3 * 10, device="cuda", dtype=torch.int32).reshape(3, 10)
    lengths = vector(prompts)
    rows = [torch.randn((sum(c), H + 2 * KV, D), device="cuda", dtype=torch.bfloat16) for c in (prompts, chunk)]
    say("a conversation")
    outs = []
    for x, counts in zip(rows, (prompts, chunk)):
        starts = vector(starts_of(counts))
        if x is rows[1]:
            lengths += vector(chunk)
        gpu.paged_append_q4(x[:, H:H + KV], x[:, H + KV:], *pools, table, lengths, starts=starts)
        held = lengths.cpu().tolist()
        whole = vector(starts_of(held))
        k, v = (torch.empty((sum(held), KV, D), device="cuda", dtype=torch.bfloat16) for _ in "kv")
        gpu.paged_read_q4(k, v, *pools, table, lengths, starts=whole)
        out = torch.empty((sum(counts), H, D), device="cuda")
        gpu.packed_attention(x[:, :H], k, v, out, starts=starts, key_starts=whole, cap=cap)
        outs.append((host(x[:, :H]), host(k), host(v), host(out), held, counts))
    for q, k, v, out, held, counts in outs:
        a, b = starts_of(counts), starts_of(held)
        for i in range(3):
            want, bound = document64(q[a[i]:a[i + 1]], k[b[i]:b[i + 1]], v[b[i]:b[i + 1]], "bf16", "f32", cap=cap)
            assert (np.abs(out[a[i]:a[i + 1]] - want) <= bound).all()
    # the newest tokens once more through the decode: the same attention, its keys not rounded to bf16
    last = torch.tensor([a - 1 for a in starts_of(chunk)[1:]], device="cuda")
    out = torch.empty((3, H, D), device="cuda")
    gpu.paged_decode_q4(rows[1][last, :H].contiguous(), out, *pools, table, lengths, cap=cap)
    k, v = (torch.empty((sum(total), KV, D), device="cuda") for _ in "kv")
    gpu.paged_read_q4(k, v, *pools, table, lengths, starts=vector(starts_of(total)))
    again = torch.empty((3, H, D), device="cuda")
    gpu.packed_attention(rows[1][last, :H].float(), k, v, again, starts=vector([0, 1, 2, 3]),
                         key_starts=vector(starts_of(total)), cap=cap)
    b = starts_of(total)
    for i in range(3):
        want, bound = document64(host(rows[1][last, :H].float())[i:i + 1], host(k)[b[i]:b[i + 1]], host(v)[b[i]:b[i + 1]],
                                 "f32", "f32", cap=cap)
        assert (np.abs(host(again)[i] - want[0]) <= bound[0]).all()
        # the decode's two-term products: four more roundings a product and a weight
        assert (np.abs(host(out)[i] - want[0]) <= 2 * bound[0]).all()
