"""A paged cache of 4-bit codes for the tests, and its operators restated in float64.

Every row of the pool that no position covers has NaN scales and codes of no
meaning, and every table entry past a sequence's last page a number that names
no page, so reading either shows."""
import numpy as np

from oracle import oracle as O
from paged_util import NORM_STEPS, TURN_STEPS, U, normed, pair_sizes, turn

BLOCK, MOST = 32, 2720.0


def encode64(x):
    """(codes 0..15 [..., dim], scales [..., dim / 32], float64) of rows: the scale by whole numbers of its unit, the
    code by comparing with the borders between the fifteen values"""
    b = np.asarray(x, np.float64)
    b = b.reshape(*b.shape[:-1], b.shape[-1] // BLOCK, BLOCK)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    e = np.frexp(top / 7)[1] - 8
    unit = np.ldexp(1.0, np.maximum(e, -24))
    n = np.floor(top / 7 / unit)
    n += 7 * n * unit < top
    scale = np.minimum(n * unit, MOST)
    code = np.full(b.shape, -7)
    for j in range(-6, 8):
        code += b >= (j - 0.5) * scale[..., None]
    code = np.where(scale[..., None] == 0, 0, code)
    code, scale = np.where(bad[..., None], 0, code), np.where(bad, np.nan, scale)
    return (code + 8).reshape(np.shape(x)), scale


def border_distance(x):
    """how far each element is from a border between two codes, in scales (of rows whose values are finite)"""
    _, scale = encode64(x)
    t = np.asarray(x, np.float64) / np.repeat(np.maximum(scale, 2.0 ** -24), BLOCK, -1)
    return np.abs(t - np.floor(t) - 0.5)


def values64(codes, scales):
    return (np.asarray(codes, np.float64) - 8) * np.repeat(np.asarray(scales, np.float64), BLOCK, -1)


class CacheQ4:
    """kind "head": the rows of one head of a page lie together, "position": the heads of one position"""

    def __init__(self, lengths, kv, page, dim, seed, kind="head", width=None, spare=2, fill=True, size=1.0):
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
        shape = (self.pages, kv, page, dim)
        self.codes = [r.integers(0, 16, shape) for _ in "kv"]
        self.scales = [np.full((*shape[:3], dim // BLOCK), np.nan) for _ in "kv"]
        for b, n in enumerate(self.lengths if fill else []):
            p = np.arange(n)
            where = self.table[b][p // page], slice(None), p % page
            for i, name in enumerate("kv"):
                if n:
                    self.codes[i][where], self.scales[i][where] = \
                        encode64(size * O.fill_normal((n, kv, dim), seed, f"{name}{b}"))

    def device(self):
        """(key codes, key scales, value codes, value scales, table, lengths) on the GPU"""
        import torch

        def pages(x):
            t = torch.from_numpy(np.ascontiguousarray(x if self.kind == "head" else x.transpose(0, 2, 1, 3))).cuda()
            return t if self.kind == "head" else t.transpose(1, 2)

        out = []
        for codes, scales in zip(self.codes, self.scales):
            out += [pages((codes[..., ::2] | codes[..., 1::2] << 4).astype(np.uint8)), pages(scales.astype(np.float16))]
        return (*out, torch.from_numpy(self.table).cuda(),
                torch.tensor(self.lengths, dtype=torch.int32, device="cuda"))

    def rows(self, b):
        """sequence b's keys and values [n][kv][dim]"""
        p = np.arange(self.lengths[b])
        at = self.table[b][p // self.page], slice(None), p % self.page
        return tuple(values64(c[at], s[at]) for c, s in zip(self.codes, self.scales))


def unpacked(codes):
    """uint8 [..., dim / 2] on the host to codes [..., dim]"""
    return np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def scored64(q, keys, values, position, gamma=None, freqs=None, interleaved=False, amplitude=1.0, scale=0.0,
             window=0, eps=1e-6, offset=0.0, cap=0.0, slopes=None, terms=3, product=0.0):
    """one token's attention in float64, its scores capped and biased, and how far fp32 work may be from it

    q [heads][dim], keys and values [n][kv][dim]; returns (out, bound), both [heads][dim]. A score's products
    (`terms` a product, each off by `product` roundings of 2^-24) add their roundings as a random walk, eight
    deviations of it counted, on top of the roundings of q's norm and rotation and the scale's; the cap (whose
    derivative is at most 1) adds four for its tanh and two products, the bias one for its product and one for the
    difference, of what it is taken from. A weight's error is its own score's less the mean of them all, two for the
    exponential's argument and result, and `product` again; the weighted sum adds as a random walk."""
    heads, dim = q.shape
    n, kv, _ = keys.shape
    begin = max(0, n - window) if window else 0
    scale = scale or 1.0 / np.sqrt(dim)
    base = normed(q, gamma, eps, offset)
    t = turn(base[None], [position], freqs, interleaved, amplitude)[0]
    size = pair_sizes(base, freqs, interleaved, amplitude)
    apart = position - np.arange(begin, n, dtype=np.float64)
    out, bound = np.zeros((heads, dim)), np.zeros((heads, dim))
    for h in range(heads):
        k, v = keys[begin:, h // (heads // kv)], values[begin:, h // (heads // kv)]
        s = k @ t[h] * scale
        e = scale * ((8 * np.sqrt(terms * dim) + 8 + product) * (np.abs(k) @ np.abs(t[h])) +
                     (TURN_STEPS + NORM_STEPS) * (np.abs(k) @ size[h]))
        if cap:
            s = cap * np.tanh(s / cap)
            e = e + 8 * np.abs(s)
        if slopes is not None:
            s = s - slopes[h] * apart
            e = e + 2 * np.abs(slopes[h] * apart)
        e = e + 4 * np.abs(s)
        w = np.exp(s - s.max())
        w /= w.sum()
        out[h] = w @ v
        a = np.abs(v)
        bound[h] = ((w * e) @ a + (w @ e) * (w @ a) + (8 * np.sqrt(terms * len(s)) + 64 + product) * (w @ a)) * U
    return out, bound
