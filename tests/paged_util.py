"""A paged cache for the tests, and the paged operators restated in float64.

Every row of the pool that no position covers holds NaN, and every table entry
past a sequence's last page a number that names no page, so reading either
shows."""
import numpy as np

from oracle import oracle as O

HALF_STEP = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}   # of a rounding, relative to the value
U = 2.0 ** -24


def rounded(x, dtype):
    """x as the values that `dtype` holds"""
    x = np.asarray(x, np.float32)
    return O.unpack_bf16(O.pack_bf16(x)).reshape(x.shape) if dtype == "bf16" else x


def turn(x, positions, freqs, interleaved=False, amplitude=1.0, sign=1.0):
    """rotary positions in float64: x [..., tokens, heads, dim], positions [tokens]"""
    x = np.array(x, np.float64)
    if freqs is None:
        return x
    n = len(freqs)
    a = np.asarray(positions, np.float64)[:, None, None] * np.asarray(freqs, np.float64)
    c, s = amplitude * np.cos(a), sign * amplitude * np.sin(a)
    lo = np.arange(0, 2 * n, 2) if interleaved else np.arange(n)
    hi = lo + 1 if interleaved else lo + n
    u, w = x[..., lo], x[..., hi]
    y = x.copy()
    y[..., lo], y[..., hi] = u * c - w * s, w * c + u * s
    return y


def pair_sizes(x, freqs, interleaved=False, amplitude=1.0):
    """|u| + |w| of each element's pair times the amplitude, |x| where nothing turns"""
    x = np.abs(np.array(x, np.float64))
    if freqs is None:
        return x
    n = len(freqs)
    lo = np.arange(0, 2 * n, 2) if interleaved else np.arange(n)
    hi = lo + 1 if interleaved else lo + n
    both = amplitude * (x[..., lo] + x[..., hi])
    x[..., lo] = x[..., hi] = both
    return x


def normed(x, gamma, eps=1e-6, offset=0.0):
    x = np.asarray(x, np.float64)
    if gamma is None:
        return x
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (np.asarray(gamma, np.float64) + offset)


# fp32 roundings of a rotated element, in units of 2^-24 |its pair|: the reduced
# angle (pi from its half step, as a turn of at most pi), cos and sin (two each,
# an ulp), their amplitude, the two products and the sum; of a norm: the sum of
# squares over at most 8 + 6 additions (halved by the root), the division, the
# root and its argument, and two products
TURN_STEPS = 10.0
NORM_STEPS = 16.0


class Cache:
    """numpy pages as torch tensors are made of them; kind "head" keeps a
    head's rows of a page together, "position" a position's heads"""

    def __init__(self, lengths, kv, page, dim, seed, kind="head", width=None, spare=2, fill=True):
        self.lengths, self.kv, self.page, self.dim, self.kind = list(lengths), kv, page, dim, kind
        need = [-(-n // page) for n in self.lengths]
        r = np.random.default_rng(seed)
        self.pages = sum(need) + spare
        order = r.permutation(self.pages)
        self.width = width or max(1, max(need, default=1))
        self.table = r.integers(self.pages, 2 ** 31 - 1, (len(need), self.width)).astype(np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.keys = np.full((self.pages, kv, page, dim), np.nan, np.float32)
        self.values = self.keys.copy()
        if fill:
            for b, n in enumerate(self.lengths):
                p = np.arange(n)
                for name, x in (("k", self.keys), ("v", self.values)):
                    x[self.table[b][p // page], :, p % page] = O.fill_normal((n, kv, dim), seed, f"{name}{b}") \
                        if n else 0.0
            self.keys, self.values = rounded(self.keys, "bf16"), rounded(self.values, "bf16")

    def device(self):
        """(key pages, value pages, table, lengths) on the GPU; the pages shaped [pages][kv][page][dim]"""
        import torch

        def pages(x):
            t = torch.from_numpy(np.ascontiguousarray(x if self.kind == "head" else x.transpose(0, 2, 1, 3)))
            t = t.cuda().to(torch.bfloat16)
            return t if self.kind == "head" else t.transpose(1, 2)

        return (pages(self.keys), pages(self.values), torch.from_numpy(self.table).cuda(),
                torch.tensor(self.lengths, dtype=torch.int32, device="cuda"))

    def rows(self, b, n=None):
        """sequence b's keys and values [n][kv][dim]"""
        p = np.arange(self.lengths[b] if n is None else n)
        at = self.table[b][p // self.page], slice(None), p % self.page
        return self.keys[at].astype(np.float64), self.values[at].astype(np.float64)


def decode64(q, keys, values, position, gamma=None, freqs=None, interleaved=False, amplitude=1.0, scale=0.0,
             window=0, eps=1e-6, offset=0.0):
    """one token's attention in float64, and how far fp32 work may be from it

    q [heads][dim], keys and values [n][kv][dim]; returns (out, bound), both
    [heads][dim]. The bound: a score's products (three terms a product) add
    their roundings as a random walk, eight deviations of it counted, on top of
    the roundings of q's norm and rotation; a weight carries its score's error
    twice (its own and the sum's), the score's own rounding and the
    exponential's; the weighted sum adds as a random walk over its terms."""
    heads, dim = q.shape
    n, kv, _ = keys.shape
    begin = max(0, n - window) if window else 0
    scale = scale or 1.0 / np.sqrt(dim)
    base = normed(q, gamma, eps, offset)
    t = turn(base[None], [position], freqs, interleaved, amplitude)[0]
    size = pair_sizes(base, freqs, interleaved, amplitude)
    out, bound = np.zeros((heads, dim)), np.zeros((heads, dim))
    for h in range(heads):
        k, v = keys[begin:, h // (heads // kv)], values[begin:, h // (heads // kv)]
        s = k @ t[h] * scale
        w = np.exp(s - s.max())
        w /= w.sum()
        out[h] = w @ v
        steps = (8 * np.sqrt(3 * dim) + 8) * (np.abs(k) @ np.abs(t[h])) + \
            (TURN_STEPS + NORM_STEPS) * (np.abs(k) @ size[h])
        es = steps.max() * scale + 2 * np.abs(s).max()
        bound[h] = (w @ np.abs(v)) * (2 * es + 8 * np.sqrt(3.0 * len(s)) + 64) * U
    return out, bound
