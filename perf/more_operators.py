"""More operators of serving, one dict per case.

    packed   attention of many documents' tokens in one call: a document mask,
             scores capped by a tanh or biased by distance, a prefix that every
             token of its document sees, a window, cached keys before the tokens
    scored   one new token's attention over bf16 pages, capped or biased likewise
    append4  new keys and values into pages of 4-bit codes, and the rows back as
             the values that the pages hold
    decode4  one new token's attention over pages of 4-bit codes

`listed` names the calls whose speed is followed, `draw` gives more of the same
ranges, and `exact` restates each in float64. With `own` false, `run` computes
them from elementary torch operations; with `own` true it calls this package.

A 4-bit row holds its elements in blocks of 32 of one scale s: the least fp16
number of at most 8 significant bits with 7 s >= max |x|, at most 2720. Element
x is the code floor(x / s + 1/2), from -7 to 7, stored plus 8, two a byte, the
first in the low half; it stands for s times the code.
"""
import math
import os
import sys

import torch

own = False

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
TYPES = {"bf16": BF16, "f32": F32}
EPS = 1e-6
BLOCK, MOST = 32, 2720.0


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # the smallest prompts: nine messages of 1 to 64 tokens in one call, fp32, scores falling with distance
        dict(name="packed-short-f32", op="packed", documents=9, low=1, high=64, empty=0, past=0, heads=12, kv_heads=12,
             dim=64, dtype="f32", out="f32", cap=0.0, distance=True, prefix=0, window=0),
        # one long prompt of an 8B-class layer with capped scores
        dict(name="packed-8192-capped", op="packed", documents=1, low=8192, high=8192, empty=0, past=0, heads=32,
             kv_heads=8, dim=128, dtype="bf16", out="bf16", cap=50.0, distance=False, prefix=0, window=0),
        # prompts of unequal lengths with a part that is seen whole (an image, an instruction), 256-wide heads, a window
        dict(name="packed-prefix-256", op="packed", documents=7, low=201, high=3001, empty=1, past=0, heads=16,
             kv_heads=4, dim=256, dtype="bf16", out="bf16", cap=0.0, distance=False, prefix=250, window=512),
        # a few new tokens of four long conversations (drafts to verify, tool answers) behind their cached keys
        dict(name="packed-chunks", op="packed", documents=4, low=5, high=27, empty=0, past=30011, heads=32, kv_heads=8,
             dim=128, dtype="bf16", out="f32", cap=0.0, distance=True, prefix=0, window=0),
        # a serving batch of a model with capped scores and 256-wide heads
        dict(name="scored-24-capped", op="scored", batch=24, low=1000, high=16001, empty=0, heads=16, kv_heads=8,
             dim=256, page=16, dtype="bf16", norm=False, rot=256, cap=50.0, distance=False, window=0, rows="head"),
        # positions by distance alone, heads of their own keys, fp32 queries, a window
        dict(name="scored-distance-f32", op="scored", batch=64, low=100, high=5000, empty=5, heads=12, kv_heads=12,
             dim=64, page=24, dtype="f32", norm=False, rot=0, cap=0.0, distance=True, window=1024, rows="head"),
        # one step of a serving batch: one token of each of 32 sequences into pages of 16
        dict(name="append4-32", op="append4", batch=32, new=1, longest=700, kv_heads=4, dim=128, page=16, dtype="bf16",
             norm=True, rot=128, rows="head", behind=0),
        # a batch of 9 prompts of unequal lengths, 8 thousand tokens in all, with rows behind the last one
        dict(name="append4-prompts", op="append4", batch=9, new=911, longest=1821, kv_heads=8, dim=128, page=64,
             dtype="bf16", norm=True, rot=128, rows="position", behind=37),
        # one conversation: one token over 4096 cached positions, 16 query and 8 key-value heads
        dict(name="decode4-1x4096", op="decode4", batch=1, low=4096, high=4096, empty=0, heads=16, kv_heads=8, dim=128,
             page=16, dtype="bf16", norm=True, rot=128, cap=0.0, distance=False, window=0, rows="head"),
        # a serving batch: 32 sequences of 1k to 32k cached positions
        dict(name="decode4-32-ragged", op="decode4", batch=32, low=1024, high=32768, empty=0, heads=32, kv_heads=4,
             dim=128, page=16, dtype="bf16", norm=True, rot=128, cap=0.0, distance=False, window=0, rows="head"),
        # many short chats in a batch padded for a captured step, capped scores: some of its places are empty
        dict(name="decode4-256-short", op="decode4", batch=256, low=1, high=700, empty=19, heads=32, kv_heads=8,
             dim=128, page=32, dtype="f32", norm=False, rot=128, cap=30.0, distance=False, window=0, rows="head"),
        # one very long document behind one question, by distance
        dict(name="decode4-1x131072", op="decode4", batch=1, low=131072, high=131072, empty=0, heads=32, kv_heads=8,
             dim=128, page=64, dtype="bf16", norm=True, rot=0, cap=0.0, distance=True, window=0, rows="position"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["packed", "packed", "scored", "append4", "decode4", "decode4"])
    dim = rng.choice([64, 96, 128, 128, 128, 192, 256])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    heads, kv = rng.choice([(12, 12), (16, 8), (32, 8), (32, 4), (16, 1), (24, 1)])
    form = dict(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), distance=rng.choice([False, False, True]))
    if op == "packed":
        # scores, times the dim, within the largest listed case's; fp32 a sixteenth of it
        room = 8192 * 8192 * 32 * 128 // 2 // (heads * dim * (16 if dtype == "f32" else 1))
        documents, past = _log(rng, 1, 60), rng.choice([0, 0, _log(rng, 1, 30000)])
        high = _log(rng, 1, 6000)
        while documents > 1 and documents * high * (high + past) > room:
            documents = (documents + 1) // 2
        while high > 1 and documents * high * (high + past) > room:
            high = (high + 1) // 2
        return dict(form, op=op, documents=documents, low=max(1, high // rng.choice([1, 3, 50])), high=high,
                    empty=rng.choice([0, 0, 1]), past=past, heads=heads, kv_heads=kv, dim=dim, dtype=dtype,
                    out=rng.choice([dtype, "f32"]), prefix=rng.choice([0, 0, _log(rng, 1, 500)]),
                    window=rng.choice([0, 0, 700]))
    common = dict(op=op, dim=dim, dtype=dtype, page=rng.choice([8, 16, 16, 24, 32, 64, 100, 256]),
                  norm=rng.choice([True, False]), rot=rng.choice([dim, dim, dim // 2, 0]),
                  rows=rng.choice(["head", "head", "position"]))
    if op == "append4":
        batch, kv = _log(rng, 1, 200), rng.choice([1, 2, 4, 8, 12])
        most = max(1, 8199 * 8 * 128 // (batch * kv * dim) // (2 if dtype == "f32" else 1))
        new = rng.choice([1, _log(rng, 1, min(2000, most))])
        return dict(common, batch=batch, new=new, kv_heads=kv, longest=2 * new + _log(rng, 1, 6000 // batch + 8),
                    behind=rng.choice([0, 0, rng.randrange(1, 60)]) if new > 1 else 0)
    batch, high = _log(rng, 1, 256), _log(rng, 1, 131072)
    room = 32 * 16896 * 4 * 128 if op == "decode4" else 24 * 8500 * 8 * 256
    while batch > 1 and batch * high * kv * dim > room:
        batch = (batch + 1) // 2
    while high > 1 and batch * high * kv * dim > room:
        high = (high + 1) // 2
    if op == "scored" and not form["cap"] and not form["distance"]:
        form["cap"] = 40.0
    return dict(common, **form, batch=batch, low=max(1, high // rng.choice([1, 2, 32])), high=high,
                empty=rng.choice([0, 0, batch // 5]), heads=heads, kv_heads=kv, window=rng.choice([0, 0, 0, 1000]))


# ------------------------------------------------------------------- inputs
def _frequencies(c):
    n = c["rot"] // 2
    return torch.tensor([1e6 ** (-j / n) for j in range(n)], dtype=F64).float() if n else None


def _slopes(heads):
    """a head's fall of the score per position: from nearly a half down to 2^-8"""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=F32)


def _spread(low, high, n):
    """n whole numbers from low to high, evenly spaced"""
    return [low + (high - low) * i // max(1, n - 1) for i in range(n)] if n > 1 else [high]


def _lengths(c):
    """a case's own lengths, of no seed: (positions of each sequence, its new tokens)"""
    if c["op"] == "packed":
        new = _spread(c["low"], c["high"], c["documents"])
        # the cached keys before each document's tokens: from half of `past` to all
        before = _spread(c["past"] // 2, c["past"], c["documents"])
        return [n + p for n, p in zip(new, before)] + [0] * c["empty"], new + [0] * c["empty"]
    if c["op"] == "append4":
        most = 2 * c["new"] - max(1, c["new"] // 9)
        new = _spread(max(1, c["new"] // 9), most, c["batch"]) if c["new"] > 1 else [1] * c["batch"]
        return [n + (c["longest"] - n) * (i + 1) // c["batch"] for i, n in enumerate(new)], new
    return _spread(c["low"], c["high"], c["batch"] - c["empty"]) + [0] * c["empty"], None


def _prefixes(c):
    """the positions that every token of a document sees"""
    lengths, _ = _lengths(c)
    return [min(c["prefix"], n) // (1 + i % 3) for i, n in enumerate(lengths)]


class _Draws:
    """seeded tensors on the GPU"""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, dtype=F32):
        return torch.randn(shape, generator=self.gen, device="cuda", dtype=F32).to(dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")

    def pool(self, c, pages):
        """pages of bf16 rows [pages][kv_heads][page][dim]; in memory the rows of one head together, or the heads of
        one position"""
        kv, s, d = c["kv_heads"], c["page"], c["dim"]
        shape = (pages, kv, s, d) if c["rows"] == "head" else (pages, s, kv, d)
        x = torch.randn(shape, generator=self.gen, device="cuda", dtype=BF16)
        return x if c["rows"] == "head" else x.transpose(1, 2)

    def table(self, c, lengths):
        """each sequence's pages, from anywhere in a pool a little larger than needed; unused entries -1"""
        need = [-(-n // c["page"]) for n in lengths]
        pages = sum(need) + 3
        order = self.order(pages)[:sum(need)].to(torch.int32)
        width = max(1, max(need))
        counts = torch.tensor(need, device="cuda")
        table = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
        table[torch.arange(width, device="cuda")[None] < counts[:, None]] = order
        return table, pages


def _starts(counts):
    return torch.tensor([0] + counts, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)


def _dense_like(x, last, dtype):
    """an empty tensor of x's leading dimensions in x's order of memory"""
    p, kv, s, _ = x.shape
    if x.is_contiguous():
        return torch.empty((p, kv, s, last), dtype=dtype, device="cuda")
    return torch.empty((p, s, kv, last), dtype=dtype, device="cuda").transpose(1, 2)


def _pages4(x):
    """(codes, scales) of a pool of bf16 rows: the pages as appends of those rows left them"""
    codes, scales = _dense_like(x, x.shape[-1] // 2, torch.uint8), _dense_like(x, x.shape[-1] // BLOCK, F16)
    step = max(1, (1 << 26) // x[0].numel())
    for at in range(0, x.shape[0], step):
        codes[at:at + step], scales[at:at + step] = _quantised(x[at:at + step].float())
    return codes, scales


def prepare(case, seed):
    c, d = case, _Draws(seed)
    t = TYPES[c["dtype"]]
    lengths, new = _lengths(c)
    s = dict(c=c)
    if c["op"] == "packed":
        n, m = sum(new), sum(lengths)
        # q, k and v as slices of the rows that one product wrote, where no cached keys come before
        H, KV, D = c["heads"], c["kv_heads"], c["dim"]
        if c["past"]:
            s["q"], kv = d.normal(n, H, D, dtype=t), d.normal(m, 2 * KV, D, dtype=t)
            s["k"], s["v"] = kv[:, :KV], kv[:, KV:]
        else:
            rows = d.normal(n, H + 2 * KV, D, dtype=t)
            s["q"], s["k"], s["v"] = rows[:, :H], rows[:, H:H + KV], rows[:, H + KV:]
        s["out"] = torch.empty((n, H, D), dtype=TYPES[c["out"]], device="cuda")
        s["starts"] = _starts(new)
        s["key_starts"] = _starts(lengths) if c["past"] else None
        s["prefix"] = torch.tensor(_prefixes(c), dtype=torch.int32, device="cuda") if c["prefix"] else None
        s["slopes"] = _slopes(H).cuda() if c["distance"] else None
        return s
    freqs = _frequencies(c)
    s["freqs"] = None if freqs is None else freqs.cuda()
    if c["op"] != "append4":
        lengths = [lengths[i] for i in d.order(len(lengths)).cpu().tolist()]
        s["slopes"] = _slopes(c["heads"]).cuda() if c["distance"] else None
    s["longest"] = max(lengths)
    s["table"], pages = d.table(c, lengths)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["gamma"] = torch.rand((c["dim"],), generator=d.gen, device="cuda") + 0.5 if c["norm"] else None
    keys, values = d.pool(c, pages), d.pool(c, pages)
    if c["op"] == "scored":
        s["keys"], s["values"] = keys, values
    else:
        s["pages"] = (*_pages4(keys), *_pages4(values))
    if c["op"] == "append4":
        s["tokens"] = sum(new)
        # k and v as slices of the rows that one product wrote
        s["kv"] = d.normal(s["tokens"] + c["behind"], 2 * c["kv_heads"], c["dim"], dtype=t)
        s["starts"] = _starts(new) if c["new"] > 1 else None
        shape = (s["tokens"] + c["behind"], c["kv_heads"], c["dim"])
        s["out"] = torch.zeros(shape, dtype=t, device="cuda"), torch.zeros(shape, dtype=t, device="cuda")
    else:
        s["q"] = d.normal(c["batch"], c["heads"], c["dim"], dtype=t)
        s["out"] = torch.empty((c["batch"], c["heads"], c["dim"]), device="cuda")
    return s


# ------------------------------------------------------------------- one pass
def _package():
    if "aigpu" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "math-utils_amd"))
    import aigpu
    return aigpu


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    c, aigpu = s["c"], _package()
    if c["op"] == "packed":
        aigpu.packed_attention(s["q"], s["k"], s["v"], s["out"], starts=s["starts"], key_starts=s["key_starts"],
                               prefix=s["prefix"], window=c["window"], cap=c["cap"], slopes=s["slopes"])
        return s["out"]
    if c["op"] == "append4":
        kv = c["kv_heads"]
        aigpu.paged_append_q4(s["kv"][:, :kv], s["kv"][:, kv:], *s["pages"], s["table"], s["lengths"],
                              starts=s["starts"], k_norm=s["gamma"], eps=EPS, freqs=s["freqs"])
        aigpu.paged_read_q4(*s["out"], *s["pages"], s["table"], s["lengths"], starts=s["starts"])
        return s["out"]
    how = dict(max_length=s["longest"], q_norm=s["gamma"], eps=EPS, freqs=s["freqs"], window=c["window"],
               cap=c["cap"], slopes=s["slopes"])
    if c["op"] == "scored":
        aigpu.paged_decode(s["q"], s["out"], s["keys"], s["values"], s["table"], s["lengths"], **how)
    else:
        aigpu.paged_decode_q4(s["q"], s["out"], *s["pages"], s["table"], s["lengths"], **how)
    return s["out"]


def _turn(x, positions, freqs):
    """x [rows][heads][dim], halves paired, rotated at positions [rows]; the angles in 64 bits"""
    if freqs is None:
        return x
    n = freqs.shape[0]
    angles = positions.to(F64)[:, None, None] * freqs.to(F64)
    cos, sin = angles.cos().to(x.dtype), angles.sin().to(x.dtype)
    a, b = x[..., :n], x[..., n:2 * n]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * n:]), -1)


def _normed(x, gamma):
    return x if gamma is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma


def _quantised(x):
    """(codes uint8 [..., dim / 2], scales fp16 [..., dim / 32]) of rows in 64 bits, or of values that 32 bits hold"""
    x = x.unflatten(-1, (-1, BLOCK)).to(F64)
    least = x.abs().amax(-1) / 7
    unit = torch.exp2((torch.floor(torch.log2(least.clamp(min=2.0 ** -60))) - 7).clamp(min=-24))
    scale = (torch.ceil(least / unit) * unit).clamp(max=MOST)
    codes = torch.floor(x / scale.masked_fill(scale == 0, 1.0)[..., None] + 0.5).clamp(-7, 7) + 8
    codes = codes.flatten(-2).to(torch.uint8)
    return codes[..., ::2] | codes[..., 1::2] << 4, scale.to(F16)


def _values(codes, scales):
    """the fp32 rows of 4-bit pages"""
    x = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
    return (x.unflatten(-1, (-1, BLOCK)) * scales.float()[..., None]).flatten(-2)


def _weighed(scores, seen, apart, c, slopes):
    """softmax weights of scores [batch][kv_heads][queries of a group][queries][keys] and their sum, over what is
    seen [batch][queries][keys]; apart: query and key positions' distance"""
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    if slopes is not None:
        scores = scores - slopes.view(1, c["kv_heads"], -1, 1, 1) * apart[:, None, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    return p, p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain(s):
    c = s["c"]
    return {"packed": _plain_packed, "append4": _plain_append}.get(c["op"], _plain_decode)(s)


def _plain_packed(s):
    c = s["c"]
    lengths, new = _lengths(c)
    n, m, docs, KV, D = max(new), max(lengths), len(new), c["kv_heads"], c["dim"]
    G = c["heads"] // KV
    starts = s["starts"].long()
    key_starts = starts if s["key_starts"] is None else s["key_starts"].long()
    counts, sizes = starts.diff(), key_starts.diff()
    rows, cols = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    # documents side by side, padded to the longest
    q = s["q"][(starts[:-1, None] + rows).clamp(max=s["q"].shape[0] - 1)].float()
    at = (key_starts[:-1, None] + cols).clamp(max=s["k"].shape[0] - 1)
    keys = s["k"][at].float().permute(0, 2, 3, 1).contiguous()
    q = q.reshape(docs, n, KV, G, D).permute(0, 2, 3, 1, 4).reshape(docs, KV, G * n, D)
    scores = (torch.matmul(q, keys) * D ** -0.5).reshape(docs, KV, G, n, m)
    place = (sizes - counts)[:, None] + rows
    apart = place[:, :, None] - cols
    seen = apart >= 0
    if s["prefix"] is not None:
        seen = seen | (cols < s["prefix"].long()[:, None])[:, None]
    if c["window"]:
        seen = seen & (apart < c["window"])
    seen = seen & (cols < sizes[:, None])[:, None]
    p, total = _weighed(scores, seen, apart.abs().float(), c, s["slopes"])
    values = s["v"][at].float().transpose(1, 2).contiguous()
    out = torch.matmul(p.reshape(docs, KV, G * n, m), values).reshape(docs, KV, G, n, D) / total
    # and packed again
    token = torch.arange(s["q"].shape[0], device="cuda")
    doc = torch.searchsorted(starts[1:].contiguous(), token, right=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(docs, n, c["heads"], D)
    s["out"].copy_(out[doc, token - starts[doc]])
    return s["out"]


def _plain_append(s):
    c, n, kv, lengths = s["c"], s["tokens"], s["c"]["kv_heads"], s["lengths"].long()
    token = torch.arange(n, device="cuda")
    if s["starts"] is None:
        seq, positions = token, lengths - 1
    else:
        starts = s["starts"].long()
        seq = torch.searchsorted(starts[1:].contiguous(), token, right=True)
        positions = lengths[seq] - starts[seq + 1] + token
    pages, rows = s["table"][seq, positions // c["page"]].long(), positions % c["page"]
    # in 64 bits: next to a border between two codes the last bit decides
    k = _turn(_normed(s["kv"][:n, :kv].to(F64), s["gamma"]), positions, s["freqs"])
    for x, (codes, scales), out in ((k, s["pages"][:2], s["out"][0]), (s["kv"][:n, kv:], s["pages"][2:], s["out"][1])):
        codes[pages, :, rows], scales[pages, :, rows] = _quantised(x)
        out[:n] = _values(codes[pages, :, rows], scales[pages, :, rows])
    return s["out"]


def _plain_decode(s):
    c = s["c"]
    B, H, KV, D = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    lengths = s["lengths"].long()
    q = _turn(_normed(s["q"].float(), s["gamma"]), (lengths - 1).clamp(min=0), s["freqs"])
    table = s["table"].long().clamp(min=0)
    if c["op"] == "scored":
        def rows(which):
            return s["keys" if which == 0 else "values"][table].transpose(1, 2).reshape(B, KV, -1, D).float()
    else:
        def rows(which):
            codes, scales = s["pages"][2 * which:2 * which + 2]
            return _values(codes[table], scales[table]).transpose(1, 2).reshape(B, KV, -1, D)
    keys = rows(0)
    at = torch.arange(keys.shape[2], device="cuda")
    apart = lengths[:, None] - 1 - at
    seen = apart >= 0
    if c["window"]:
        seen = seen & (apart < c["window"])
    q = q.reshape(B, KV, H // KV, D).transpose(2, 3).contiguous()
    scores = (torch.matmul(keys, q) * D ** -0.5).transpose(2, 3)[:, :, :, None]
    del keys
    p, total = _weighed(scores, seen[:, None], apart.abs().float()[:, None], c, s["slopes"])
    return (torch.matmul(p[:, :, :, 0].contiguous(), rows(1)) / total[:, :, :, 0]).reshape(B, H, D)


# ------------------------------------------------------------------- the work
def _pairs(c):
    """the (query, key) pairs of a packed case that see each other, and the keys that any query sees"""
    pairs, (lengths, new) = 0, _lengths(c)
    for n, q, prefix in zip(lengths, new, _prefixes(c)):
        for i in range(n - q, n):
            first = max(0, i + 1 - c["window"]) if c["window"] else 0
            pairs += max(i + 1, prefix) - first
    return pairs


def work(case):
    c = case
    e = 2 if c["dtype"] == "bf16" else 4
    lengths, new = _lengths(c)
    D = c["dim"]
    if c["op"] == "packed":
        o = 2 if c["out"] == "bf16" else 4
        rows = sum(new) * c["heads"] * D
        seen = sum(min(n, q + c["window"] - 1) if c["window"] and q else n if q else 0 for n, q in zip(lengths, new))
        return {"bytes": rows * (e + o) + 2 * seen * c["kv_heads"] * D * e,
                "flops": 4 * _pairs(c) * c["heads"] * D}
    row4 = D / 2 + D / 16
    if c["op"] == "append4":
        rows = 2 * sum(new) * c["kv_heads"]
        return {"bytes": rows * (2 * D * e + 2 * row4), "flops": 10 * rows * D}
    seen = sum(min(x, c["window"]) if c["window"] else x for x in lengths)
    rows = c["batch"] * c["heads"] * D
    per = 2 * row4 if c["op"] == "decode4" else 4 * D
    return {"bytes": per * seen * c["kv_heads"] + rows * (e + 4) + 4 * (seen // c["page"] + c["batch"]),
            "flops": 4 * seen * c["heads"] * D}


# ------------------------------------------------------------------- in 64 bits
def _exact_turn(x, p, freqs):
    """x [..., dim] in float64 as complex pairs times e^{i p f}; p broadcasts over x[..., 0]"""
    if freqs is None:
        return x
    n = freqs.shape[0]
    turn = torch.polar(torch.ones_like(p[..., None] * freqs.to(F64)), p[..., None] * freqs.to(F64))
    z = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()) * turn
    return torch.cat((z.real, z.imag, x[..., 2 * n:]), -1)


def _exact_norm(x, gamma):
    if gamma is None:
        return x
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * gamma.to(F64)


def _exact_round(x):
    """rows in float64 as the values that their 4-bit codes stand for: the scale by its significand, the code as the
    nearest of the fifteen values (the upper one of two)"""
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    top = b.abs().amax(-1)
    _, e = torch.frexp(top / 7)                      # its significand in [1/2, 1)
    e = (e - 8).clamp(min=-24, max=100).long()       # that of its eighth bit, or 2^-24's
    unit = torch.tensor([math.ldexp(1.0, i) for i in range(-24, 101)], dtype=F64, device="cuda")[e + 24]
    scale = (torch.ceil(top / 7 / unit) * unit).clamp(max=MOST)
    code = torch.zeros_like(b, dtype=F64) - 7
    for j in range(-6, 8):
        code += (b >= (j - 0.5) * scale[..., None]).to(F64)
    return (code * scale[..., None]).reshape(x.shape)


def _exact_attention(q, k, v, where, c, slopes, prefix):
    """q [queries][heads][dim] at positions `where` over k, v [keys][kv_heads][dim], all float64"""
    G = c["heads"] // c["kv_heads"]
    out = torch.zeros_like(q)
    j = torch.arange(k.shape[0], device="cuda", dtype=F64)
    gap = where[:, None] - j
    hidden = (gap < 0) & ~(j < prefix)
    if c["window"]:
        hidden |= gap >= c["window"]
    for h in range(c["heads"]):
        x = q[:, h] @ k[:, h // G].T / math.sqrt(c["dim"])
        if c["cap"]:
            x = torch.tanh(x / c["cap"]) * c["cap"]
        if slopes is not None:
            x -= gap.abs() * slopes[h].to(F64)
        x[hidden] = -math.inf
        out[:, h] = torch.nan_to_num(x.softmax(-1)) @ v[:, h // G]
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "packed":
        lengths, new = _lengths(c)
        out, q0, k0 = torch.zeros(s["out"].shape, dtype=F64, device="cuda"), 0, 0
        for n, q, prefix in zip(lengths, new, _prefixes(c)):
            if q:
                where = torch.arange(n - q, n, device="cuda", dtype=F64)
                out[q0:q0 + q] = _exact_attention(s["q"][q0:q0 + q].to(F64), s["k"][k0:k0 + n].to(F64),
                                                  s["v"][k0:k0 + n].to(F64), where, c, s["slopes"], prefix)
            q0, k0 = q0 + q, k0 + n
        return out
    lengths = s["lengths"].cpu().tolist()
    if c["op"] == "append4":
        kv, (_, new), first = c["kv_heads"], _lengths(c), 0
        k, v = (torch.zeros(x.shape, dtype=F64, device="cuda") for x in s["out"])
        for n, q in zip(lengths, new):
            p = torch.arange(n - q, n, device="cuda", dtype=F64)[:, None]
            x = s["kv"][first:first + q].to(F64)
            k[first:first + q] = _exact_round(_exact_turn(_exact_norm(x[:, :kv], s["gamma"]), p, s["freqs"]))
            v[first:first + q] = _exact_round(x[:, kv:])
            first += q
        return k, v
    out = torch.zeros((c["batch"], c["heads"], c["dim"]), dtype=F64, device="cuda")
    table = s["table"].cpu()
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        pages = table[b][:-(-n // c["page"])].long().cuda()
        begin = max(0, n - c["window"]) if c["window"] else 0

        def rows(which):
            if c["op"] == "scored":
                x = s["keys" if which == 0 else "values"][pages].to(F64)
            else:
                codes, scales = (t[pages] for t in s["pages"][2 * which:2 * which + 2])
                x = torch.empty((*codes.shape[:-1], c["dim"]), dtype=F64, device="cuda")
                x[..., 0::2], x[..., 1::2] = codes % 16, codes // 16
                x = (x - 8) * scales.to(F64).repeat_interleave(BLOCK, -1)
            return x.permute(0, 2, 1, 3).reshape(-1, c["kv_heads"], c["dim"])[begin:n]

        last = torch.tensor([float(n - 1)], dtype=F64, device="cuda")
        q = _exact_turn(_exact_norm(s["q"][b].to(F64), s["gamma"]), last, s["freqs"])
        out[b] = _exact_attention(q[None], rows(0), rows(1), last - begin, c, s["slopes"], 0)[0]
    return out
