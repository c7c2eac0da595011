"""A bound of the paged decode's error that a lost term of its products exceeds,
and those products restated in numpy with fewer terms.

The operator cuts an fp32 query (and each softmax weight) into three bf16 terms
of 8 bits whose sum it is, so its products are fp32's. Without the third term a
query element is off by 2^-16 of itself, some 200 units U = 2^-24 of a score's
size, where fp32's own roundings come to about ten. decode64's bound
(paged_util.py) sums the products' sizes, and so is wider than either."""
import numpy as np

from paged_util import U, normed, pair_sizes, turn


def tight64(q, keys, values, position, gamma=None, freqs=None, interleaved=False, amplitude=1.0, scale=0.0, window=0,
            eps=1e-6, offset=0.0):
    """one token's attention in float64 and a bound of fp32 work on it, both [heads][dim]; arguments as decode64's

    Roundings are counted as deviations, eight of which bound their sum. A
    rounding is uniform within half a step, at most U of its value: U / sqrt(3)
    a deviation. A sum of n products in one order rounds partial sums that grow
    like their root: U sqrt(n / 6) of the root of the products' squares. Of a
    score: that sum over the terms of 8 bits that lead (the lower ones' sums are
    2^-8 of it), the scale's rounding of each element (1), two to four more each
    where elements are normed or turned (cos and sin to 2.5 steps, two products,
    a sum). Of a weight: its score's, the exponential's, and those of the
    running maximum's and the joins' factors (7 in all), an argument's (2 of
    it). Weights matter by how far their value is from the average. All scores
    alike: the scale, its constant, the norm's root and mean (12 of each
    score's distance from the average one); all weights up to a place alike: a
    factor (8). Then the weighted sum, 3 n roundings (a term's products each) of
    partial sums no larger than their end and their root together, the sum of
    weights, n of them, and the quotient (4)."""
    heads, dim = q.shape
    n, kv, _ = keys.shape
    begin = max(0, n - window) if window else 0
    scale = scale or 1.0 / np.sqrt(dim)
    base = normed(q, gamma, eps, offset)
    t = turn(base[None], [position], freqs, interleaved, amplitude)[0]
    size = pair_sizes(base, freqs, interleaved, amplitude)
    each = 1.0 + (4.0 if freqs is not None else 0.0) + (2.0 if gamma is not None else 0.0)
    out, bound = np.zeros((heads, dim)), np.zeros((heads, dim))
    for h in range(heads):
        k, v = keys[begin:, h // (heads // kv)], values[begin:, h // (heads // kv)]
        s = k @ t[h] * scale
        w = np.exp(s - s.max())
        w /= w.sum()
        out[h] = w @ v
        root = np.sqrt((k * k) @ (t[h] * t[h])) * scale
        rough = np.sqrt((k * k) @ (size[h] * size[h])) * scale
        es = np.sqrt(dim / 6.0) * root + each * rough
        ew = es + 7.0 + 2.0 * np.abs(s - s.max())
        off = v - out[h]
        walk = 8 * np.sqrt(((w * ew)[:, None] ** 2 * off ** 2).sum(0))
        alike = 12 * (w * np.abs(s - w @ s)) @ np.abs(off) + 8 * w @ np.abs(off)
        sums = 8 * (np.sqrt(3 * len(s) / 6.0) * (np.sqrt((w * w) @ (v * v)) + np.abs(out[h])) +
                    np.sqrt(len(s) / 6.0) * np.abs(out[h]))
        bound[h] = (walk + alike + sums + 4 * np.abs(out[h])) * U
    return out, bound


def terms(x, count):
    """fp32 x as the sum of `count` terms of 8 bits, each cut off: what is left after the third is nothing"""
    rest, out = np.asarray(x, np.float32).copy(), []
    for _ in range(count):
        out.append((rest.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32))
        rest = rest - out[-1]
    return out


def restated(q, keys, values, query_terms, weight_terms, scale=0.0):
    """the decode of fp32 queries [heads][dim] in fp32, with so many terms of the queries and of the weights"""
    heads, dim = q.shape
    kv = keys.shape[1]
    factor = np.float32((scale or 1.0 / np.sqrt(dim)) * 1.4426950408889634)
    out = np.zeros((heads, dim), np.float32)
    for h in range(heads):
        k, v = (x[:, h // (heads // kv)].astype(np.float32) for x in (keys, values))
        s = np.zeros(len(k), np.float32)
        for part in terms(np.asarray(q[h], np.float32) * factor, query_terms)[::-1]:
            for d in range(dim):
                s = s + k[:, d] * part[d]
        p = np.exp2((s - s.max()).astype(np.float32))
        acc = np.zeros(dim, np.float32)
        for part in terms(p, weight_terms)[::-1]:
            for j in range(len(k)):
                acc = acc + part[j] * v[j]
        out[h] = acc / p.sum(dtype=np.float32)
    return out
