"""The operators of serving from a paged key-value cache, one dict per case.

    rotary   rotary positions of query or key heads: both pair layouts, part
             of the head, frequencies scaled for long contexts, forward and
             backward (the transposed rotation)
    append   new keys and values of a batch of sequences into a paged cache,
             the keys normed and rotated on the way
    decode   one new token's attention over each sequence's pages

`listed` names the calls whose speed is followed, `draw` gives more of the same
ranges, and `exact` restates each in float64. With `own` false, `run` computes
them from elementary torch operations; with `own` true it calls this package.
"""
import math
import os
import sys

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bf16": BF16, "f32": F32}
EPS = 1e-6


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # the smallest call: one token's 32 query heads, as one step of one conversation rotates them
        dict(name="rotary-1", op="rotary", tokens=1, heads=32, dim=128, rot=128, interleaved=False, dtype="bf16",
             scaling="none", backward=False),
        # a long prompt's query heads of an 8B-class layer, in place of what a prefill does on load
        dict(name="rotary-8192", op="rotary", tokens=8192, heads=32, dim=128, rot=128, interleaved=False, dtype="bf16",
             scaling="linear", backward=False),
        # the gradient of a partly rotated head with interleaved pairs, fp32, a batch of an odd number of tokens
        dict(name="rotary-backward-1999", op="rotary", tokens=1999, heads=40, dim=192, rot=64, interleaved=True,
             dtype="f32", scaling="yarn", backward=True),
        # one step of a serving batch: one token of each of 32 sequences into pages of 16
        dict(name="append-32", op="append", batch=32, new=1, longest=700, kv_heads=4, dim=128, page=16, dtype="bf16",
             norm=True, rot=128, interleaved=False, scaling="none", rows="head", behind=0),
        # a batch of 9 prompts of unequal lengths, 8 thousand tokens in all, with rows behind the last one
        dict(name="append-prompts", op="append", batch=9, new=911, longest=1821, kv_heads=8, dim=128, page=64,
             dtype="bf16", norm=True, rot=128, interleaved=False, scaling="linear", rows="head", behind=37),
        # fp32 rows of a partly rotated 64-wide head into odd pages that keep a position's heads together
        dict(name="append-f32-odd", op="append", batch=5, new=333, longest=2000, kv_heads=12, dim=64, page=24,
             dtype="f32", norm=False, rot=32, interleaved=True, scaling="yarn", rows="position", behind=0),
        # one conversation: one token over 4096 cached positions, 16 query and 8 key-value heads
        dict(name="decode-1x4096", op="decode", batch=1, low=4096, high=4096, empty=0, heads=16, kv_heads=8, dim=128,
             page=16, dtype="bf16", norm=True, rot=128, interleaved=False, scaling="none", window=0, rows="head"),
        # a serving batch: 32 sequences of 1k to 32k cached positions
        dict(name="decode-32-ragged", op="decode", batch=32, low=1024, high=32768, empty=0, heads=32, kv_heads=4,
             dim=128, page=16, dtype="bf16", norm=True, rot=128, interleaved=False, scaling="none", window=0,
             rows="head"),
        # many short chats in a batch padded for a captured step: some of its places are empty
        dict(name="decode-256-short", op="decode", batch=256, low=1, high=700, empty=19, heads=32, kv_heads=8, dim=128,
             page=32, dtype="bf16", norm=False, rot=128, interleaved=False, scaling="linear", window=0, rows="head"),
        # one very long document behind one question
        dict(name="decode-1x131072", op="decode", batch=1, low=131072, high=131072, empty=0, heads=32, kv_heads=8,
             dim=128, page=64, dtype="bf16", norm=True, rot=128, interleaved=False, scaling="yarn", window=0,
             rows="position"),
        # heads of their own keys, 64 wide, fp32 queries, a sliding window and pages of 24
        dict(name="decode-window-f32", op="decode", batch=24, low=300, high=9000, empty=0, heads=12, kv_heads=12,
             dim=64, page=24, dtype="f32", norm=False, rot=32, interleaved=True, scaling="none", window=1024,
             rows="head"),
        # one key-value head of 256 under 16 query heads
        dict(name="decode-one-kv-head", op="decode", batch=16, low=2000, high=6001, empty=0, heads=16, kv_heads=1,
             dim=256, page=16, dtype="bf16", norm=False, rot=128, interleaved=False, scaling="none", window=0,
             rows="position"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "decode", "decode"])
    dim = rng.choice([64, 96, 128, 128, 128, 192, 256])
    rot = rng.choice([dim, dim, dim // 2, 2 * rng.randrange(1, dim // 2)])
    common = dict(op=op, dim=dim, rot=rot, interleaved=rng.choice([False, False, True]),
                  dtype=rng.choice(["bf16", "bf16", "f32"]), scaling=rng.choice(["none", "linear", "yarn"]))
    if op == "rotary":
        heads = rng.choice([1, 8, 12, 32, 40, 128])
        most = 8192 * 32 * 128 // (heads * dim) // (2 if common["dtype"] == "f32" else 1)
        return dict(common, tokens=_log(rng, 1, min(16384, most)), heads=heads, backward=rng.choice([False, False, True]))
    common.update(page=rng.choice([8, 16, 16, 24, 32, 64, 100, 256]), norm=rng.choice([True, False]),
                  rows=rng.choice(["head", "head", "position"]))
    if op == "append":
        batch, kv = _log(rng, 1, 200), rng.choice([1, 2, 4, 8, 12])
        most = max(1, 8199 * 8 * 128 // (batch * kv * dim) // (2 if common["dtype"] == "f32" else 1))
        new = rng.choice([1, _log(rng, 1, min(2000, most))])
        return dict(common, batch=batch, new=new, kv_heads=kv, longest=2 * new + _log(rng, 1, 6000 // batch + 8),
                    behind=rng.choice([0, 0, rng.randrange(1, 60)]) if new > 1 else 0)
    heads, kv = rng.choice([(12, 12), (16, 8), (32, 8), (32, 4), (16, 1), (24, 1)])
    batch, high = _log(rng, 1, 256), _log(rng, 1, 131072)
    while batch > 1 and batch * high * kv * dim > 32 * 16896 * 4 * 128:
        batch = (batch + 1) // 2
    while high > 1 and batch * high * kv * dim > 32 * 16896 * 4 * 128:
        high = (high + 1) // 2
    return dict(common, batch=batch, low=max(1, high // rng.choice([1, 2, 32])), high=high,
                empty=rng.choice([0, 0, batch // 5]), heads=heads, kv_heads=kv,
                window=rng.choice([0, 0, 0, 1000]))


# ------------------------------------------------------------------- inputs
def _frequencies(c):
    """(fp32 frequencies, the amplitude of cos and sin) of a case's scaling:
    base 1e6; linear: positions in a quarter; yarn: the slow pairs in an
    eighth, the fast ones as they are, a ramp between (trained on 4096)"""
    n, base = c["rot"] // 2, 1e6
    f = torch.tensor([base ** (-j / n) for j in range(n)], dtype=F64)
    if c["scaling"] == "linear":
        return (f / 4).float(), 1.0
    if c["scaling"] == "yarn":
        at = [2 * n * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        low, high = max(0, math.floor(at[0])), min(2 * n - 1, math.ceil(at[1]))
        ramp = ((torch.arange(n, dtype=F64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return (f / 8 * ramp + f * (1 - ramp)).float(), 0.1 * math.log(8.0) + 1.0
    return f.float(), 1.0


def _spread(low, high, n):
    """n whole numbers from low to high, evenly spaced"""
    return [low + (high - low) * i // max(1, n - 1) for i in range(n)] if n > 1 else [high]


def _counts(c):
    """the new tokens of each sequence of an append: one each, or spread round `new`"""
    return _spread(max(1, c["new"] // 9), 2 * c["new"] - max(1, c["new"] // 9), c["batch"]) if c["new"] > 1 \
        else [1] * c["batch"]


def _lengths(c):
    """the cached positions of each sequence, a case's own and of no seed: (lengths, new tokens)"""
    if c["op"] == "append":
        new = _counts(c)
        return [n + (c["longest"] - n) * (i + 1) // c["batch"] for i, n in enumerate(new)], new
    live = c["batch"] - c["empty"]
    return _spread(c["low"], c["high"], live) + [0] * c["empty"], None


class _Draws:
    """seeded tensors on the GPU"""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, dtype=F32):
        return torch.randn(shape, generator=self.gen, device="cuda", dtype=F32).to(dtype)

    def shuffled(self, values):
        at = torch.randperm(len(values), generator=self.gen, device="cuda").cpu().tolist()
        return [values[i] for i in at]

    def pool(self, c, pages):
        """pages of bf16 rows; the rows of one key-value head together, or the heads of one position"""
        kv, s, d = c["kv_heads"], c["page"], c["dim"]
        shape = (pages, kv, s, d) if c["rows"] == "head" else (pages, s, kv, d)
        x = torch.randn(shape, generator=self.gen, device="cuda", dtype=BF16)
        return x if c["rows"] == "head" else x.transpose(1, 2)

    def table(self, c, lengths):
        """each sequence's pages, from anywhere in a pool a little larger than needed; unused entries -1"""
        need = [-(-n // c["page"]) for n in lengths]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=self.gen, device="cuda")[:sum(need)].to(torch.int32)
        width = max(1, max(need))
        counts = torch.tensor(need, device="cuda")
        table = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
        table[torch.arange(width, device="cuda")[None] < counts[:, None]] = order
        return table, pages


def prepare(case, seed):
    c, d = case, _Draws(seed)
    freqs, amplitude = _frequencies(c)
    s = dict(c=c, freqs=freqs.cuda(), amplitude=amplitude)
    t = TYPES[c["dtype"]]
    if c["op"] == "rotary":
        s["x"] = d.normal(c["tokens"], c["heads"], c["dim"], dtype=t)
        # the tokens of a chunk that starts somewhere in a long context
        first = int(torch.randint(0, 100000, (1,), generator=d.gen, device="cuda"))
        s["positions"] = torch.arange(first, first + c["tokens"], dtype=torch.int32, device="cuda")
        s["out"] = torch.empty_like(s["x"])
        return s
    lengths, new = _lengths(c)
    if c["op"] == "decode":
        lengths = d.shuffled(lengths)
    s["longest"] = max(lengths)
    s["table"], pages = d.table(c, lengths)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["keys"], s["values"] = d.pool(c, pages), d.pool(c, pages)
    s["gamma"] = torch.rand((c["dim"],), generator=d.gen, device="cuda") + 0.5 if c["norm"] else None
    if c["op"] == "append":
        s["tokens"] = sum(new)
        rows = s["tokens"] + c["behind"]
        # k and v as slices of the rows that one product wrote
        s["kv"] = d.normal(rows, 2 * c["kv_heads"], c["dim"], dtype=t)
        s["starts"] = None
        if c["new"] > 1:
            s["starts"] = torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
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
    if c["op"] == "rotary":
        aigpu.rotary(s["x"], s["out"], s["freqs"], positions=s["positions"], interleaved=c["interleaved"],
                     amplitude=s["amplitude"], backward=c["backward"])
        return s["out"]
    if c["op"] == "append":
        kv = c["kv_heads"]
        aigpu.paged_append(s["kv"][:, :kv], s["kv"][:, kv:], s["keys"], s["values"], s["table"], s["lengths"],
                           starts=s["starts"], k_norm=s["gamma"], eps=EPS, freqs=s["freqs"],
                           interleaved=c["interleaved"], amplitude=s["amplitude"])
        return s["keys"], s["values"]
    aigpu.paged_decode(s["q"], s["out"], s["keys"], s["values"], s["table"], s["lengths"], max_length=s["longest"],
                       q_norm=s["gamma"], eps=EPS, freqs=s["freqs"], interleaved=c["interleaved"],
                       amplitude=s["amplitude"], window=c["window"])
    return s["out"]


def _turn(x, positions, s, backward=False):
    """x [rows][heads][dim] in fp32, rotated at positions [rows]; the angles in 64 bits"""
    c, rot = s["c"], s["c"]["rot"]
    angles = positions.to(F64)[:, None, None] * s["freqs"].to(F64)
    cos, sin = (angles.cos() * s["amplitude"]).float(), (angles.sin() * s["amplitude"]).float()
    if backward:
        sin = -sin
    if c["interleaved"]:
        a, b = x[..., :rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return turned if rot == c["dim"] else torch.cat((turned, x[..., rot:]), -1)


def _normed(x, gamma):
    return x if gamma is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma


def _plain(s):
    c = s["c"]
    if c["op"] == "rotary":
        return _turn(s["x"].float(), s["positions"], s, c["backward"]).to(s["x"].dtype)
    if c["op"] == "append":
        n, kv, lengths = s["tokens"], c["kv_heads"], s["lengths"].long()
        token = torch.arange(n, device="cuda")
        if s["starts"] is None:
            seq, positions = token, lengths - 1
        else:
            starts = s["starts"].long()
            seq = torch.searchsorted(starts[1:].contiguous(), token, right=True)
            positions = lengths[seq] - starts[seq + 1] + token
        pages, rows = s["table"][seq, positions // c["page"]].long(), positions % c["page"]
        k = _turn(_normed(s["kv"][:n, :kv].float(), s["gamma"]), positions, s)
        s["keys"][pages, :, rows] = k.to(BF16)
        s["values"][pages, :, rows] = s["kv"][:n, kv:].to(BF16)
        return s["keys"], s["values"]
    B, H, KV, D = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    lengths = s["lengths"].long()
    q = _turn(_normed(s["q"].float(), s["gamma"]), (lengths - 1).clamp(min=0), s)
    table = s["table"].long().clamp(min=0)
    keys = s["keys"][table].transpose(1, 2).reshape(B, KV, -1, D).float()
    at = torch.arange(keys.shape[2], device="cuda")
    seen = at < lengths[:, None]
    if c["window"]:
        seen &= at >= lengths[:, None] - c["window"]
    q = q.reshape(B, KV, H // KV, D).transpose(2, 3).contiguous()
    scores = torch.matmul(keys, q) * D ** -0.5
    del keys
    scores = scores.transpose(2, 3).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    values = s["values"][table].transpose(1, 2).reshape(B, KV, -1, D).float()
    out = torch.matmul(p.contiguous(), values) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.reshape(B, H, D)


# ------------------------------------------------------------------- the work
def work(case):
    c = case
    e = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "rotary":
        n = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * e + 4 * c["tokens"] + 2 * c["rot"], "flops": 3 * n}
    lengths, new = _lengths(c)
    if c["op"] == "append":
        n = sum(new) * c["kv_heads"] * c["dim"]
        return {"bytes": 2 * n * (e + 2) + 4 * sum(-(-x // c["page"]) for x in new) + 8 * c["batch"], "flops": 6 * n}
    seen = sum(min(x, c["window"]) if c["window"] else x for x in lengths)
    rows = c["batch"] * c["heads"] * c["dim"]
    return {"bytes": 4 * seen * c["kv_heads"] * c["dim"] + rows * (e + 4) + 4 * (seen // c["page"] + c["batch"]),
            "flops": 4 * seen * c["heads"] * c["dim"]}


# ------------------------------------------------------------------- in 64 bits
def _exact_turn(x, p, freqs, amplitude, rot, interleaved, sign=1.0):
    """x [..., dim] in float64 as complex pairs times amplitude e^{i sign p f}; p broadcasts over x[..., 0]"""
    turn = torch.polar(torch.full_like(p[..., None] * freqs, amplitude), sign * p[..., None] * freqs)
    y = x.clone()
    at = torch.arange(0, rot, 2, device=x.device) if interleaved else torch.arange(rot // 2, device=x.device)
    far = at + 1 if interleaved else at + rot // 2
    z = torch.complex(x[..., at], x[..., far]) * turn
    y[..., at], y[..., far] = z.real, z.imag
    return y


def exact(case, seed):
    c, s = case, prepare(case, seed)
    f, A, D = s["freqs"].to(F64), s["amplitude"], c["dim"]

    def norm(x):
        if s["gamma"] is None:
            return x
        return x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * s["gamma"].to(F64)

    if c["op"] == "rotary":
        return _exact_turn(s["x"].to(F64), s["positions"].to(F64)[:, None], f, A, c["rot"], c["interleaved"],
                           -1.0 if c["backward"] else 1.0)
    lengths = s["lengths"].cpu().tolist()
    table = s["table"].cpu()
    if c["op"] == "append":
        kv, (_, new) = c["kv_heads"], _lengths(c)
        keys, values, first = s["keys"].to(F64), s["values"].to(F64), 0
        for b, n in enumerate(new):
            p = torch.arange(lengths[b] - n, lengths[b])
            pages, rows = table[b][p // c["page"]].long().cuda(), (p % c["page"]).cuda()
            rowsin = s["kv"][first:first + n].to(F64)
            keys[pages, :, rows] = _exact_turn(norm(rowsin[:, :kv]), p.to(F64).cuda()[:, None], f, A, c["rot"],
                                               c["interleaved"])
            values[pages, :, rows] = rowsin[:, kv:]
            first += n
        return keys, values
    G = c["heads"] // c["kv_heads"]
    out = torch.zeros((c["batch"], c["heads"], D), dtype=F64, device="cuda")
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        last = torch.tensor([n - 1.0], dtype=F64, device="cuda")
        q = _exact_turn(norm(s["q"][b].to(F64)), last, f, A, c["rot"], c["interleaved"])
        pages = table[b][:-(-n // c["page"])].long().cuda()
        begin = max(0, n - c["window"]) if c["window"] else 0
        for h in range(c["kv_heads"]):
            k = s["keys"][pages, h].reshape(-1, D)[begin:n].to(F64)
            v = s["values"][pages, h].reshape(-1, D)[begin:n].to(F64)
            w = (q[h * G:(h + 1) * G] @ k.T / math.sqrt(D)).softmax(-1)
            out[b, h * G:(h + 1) * G] = w @ v
    return out
