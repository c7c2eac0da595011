"""Attention of packed documents restated in float64, and how far the kernel's types may be from it."""
import numpy as np

from paged_util import U

# half a step of a weight, relative to it
WEIGHT = {("bf16", "bf16"): 2.0 ** -8, ("bf16", "f32"): 0.0, ("f32", "f32"): 0.0, ("f32", "bf16"): 0.0}
OUT = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def document64(q, k, v, dtype, out, prefix=0, window=0, cap=0.0, slopes=None, scale=0.0):
    """one document in float64: q [tokens][heads][dim], k and v [keys][kv][dim]; returns (out, bound)

    A score's products are exact or round once, and add as a random walk (eight deviations); the cap, the bias, the
    weights' exponential and the weighted sum add their roundings as scored64 says. A rounded weight moves the result
    by its half step of the value's distance from the result, as the sum adds what was rounded."""
    n, heads, dim = q.shape
    m, kv, _ = k.shape
    scale = scale or 1.0 / np.sqrt(dim)
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    at = np.arange(m - n, m)[:, None]
    j = np.arange(m)
    seen = (j <= at) | (j < prefix)
    if window:
        seen &= at - j < window
    res, bound = np.zeros((n, heads, dim)), np.zeros((n, heads, dim))
    some = seen.any(1)
    if not some.any():
        return res, bound
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        s = q[:, h] @ kh.T * scale
        e = scale * (8 * np.sqrt(dim) + 8) * (np.abs(q[:, h]) @ np.abs(kh).T)
        if cap:
            s = cap * np.tanh(s / cap)
            e = e + 8 * np.abs(s)
        if slopes is not None:
            bias = slopes[h] * np.abs(at - j)
            s = s - bias
            e = e + 2 * np.abs(bias)
        e = e + 4 * np.abs(s)
        s = np.where(seen, s, -np.inf)
        top = s.max(1, keepdims=True)
        w = np.exp(s - np.where(np.isfinite(top), top, 0.0))
        total = w.sum(1, keepdims=True)
        w = w / np.where(total > 0, total, 1.0)
        e = np.where(seen, e, 0.0)
        res[:, h] = w @ vh
        a = np.abs(vh)
        bound[:, h] = ((w * e) @ a + (w * e).sum(1, keepdims=True) * (w @ a) + (8 * np.sqrt(2.0 * m) + 64) * (w @ a)) * U
        step = WEIGHT[dtype, out]
        if step:
            off = np.abs(vh[None] - res[:, h][:, None])
            bound[:, h] += 1.02 * step * np.einsum("ij,ijd->id", w, off)
        bound[:, h] += OUT[out] * np.abs(res[:, h])
    return res, bound
