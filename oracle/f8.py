"""e4m3 with a scale per block of 128, its product, and tokens sorted by expert and
back, restated in numpy (oracle; test infrastructure only).

Codes and scales are defined to the last bit: a division and a rounding per
value.  Products, sums and gradients are given in fp64, with a bound of what
their fp32 evaluation may differ by.
"""
import numpy as np

from .formats import F32, e4m3_decode, e4m3_encode
from .q8 import MIN_AMAX


def _codes(v, axes):
    """Codes (u8) and scales (kept dimensions) of fp32 values, one scale over `axes`."""
    bad = ~np.isfinite(v).all(axes, keepdims=True)
    v = np.where(bad, F32(0), v)
    s = np.maximum(np.abs(v).max(axes, keepdims=True), MIN_AMAX) / F32(448)
    return e4m3_encode(v / s, saturate=True).astype(np.uint8), np.where(bad, F32(np.nan), s)


def quantize_rows(v):
    """(codes u8 [M, H], scales fp32 [M, ceil(H/128)]) of fp32 rows."""
    v = np.asarray(v, F32)
    parts = [_codes(v[:, b:b + 128], (1,)) for b in range(0, v.shape[1], 128)]
    return np.concatenate([q for q, _ in parts], 1), np.concatenate([s for _, s in parts], 1)


def quantize_weight(w):
    """(codes u8 [N, K], scales fp32 [ceil(N/128), ceil(K/128)]) of an fp32 matrix."""
    w = np.asarray(w, F32)
    n, k = w.shape
    q, s = np.empty((n, k), np.uint8), np.empty((-(-n // 128), -(-k // 128)), F32)
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            at = slice(128 * i, 128 * i + 128), slice(128 * j, 128 * j + 128)
            q[at], one = _codes(w[at], (0, 1))
            s[i, j] = one[0, 0]
    return q, s


def linear(xq, xs, wq, ws, bias=None, cut=False):
    """(y, bound) in fp64: the product of u8 codes, and how far an fp32 evaluation in blocks may be from it.

    A block of 128: products of two e4m3 values are exact in fp32 (8 bits); 127 additions, each off by at most a
    unit of the last place, 2^-23 (a matrix core may cut rather than round).  Both scales' product: 2^-24.  Then an
    fma per block, and at most 8 partial sums of a split over K: 2^-24 each of a sum that is at most the sum of the
    magnitudes.  The bias: 2^-24 of the result.

    cut: the products are the fp8 instruction's, which adds eight neighbours at a time, each cut towards zero to
    2^-13 of the power of two of the largest: seven of them lose less than that each, and the largest is at most the
    product of the eight's largest factors."""
    x, w = e4m3_decode(xq).astype(np.float64), e4m3_decode(wq).astype(np.float64)
    xs, ws = np.asarray(xs, np.float64), np.asarray(ws, np.float64)
    y, mag = 0.0, 0.0
    blocks = xs.shape[1]

    def largest(a):
        return np.abs(np.pad(a, ((0, 0), (0, -a.shape[1] % 8)))).reshape(a.shape[0], -1, 8).max(-1)
    with np.errstate(invalid="ignore"):
        for b in range(blocks):
            at = slice(128 * b, 128 * b + 128)
            f = xs[:, b:b + 1] * np.repeat(ws[:, b], 128)[None, :w.shape[0]]
            y = y + (x[:, at] @ w[:, at].T) * f
            mag = mag + (np.abs(x[:, at]) @ np.abs(w[:, at]).T) * np.abs(f) * (127 * 2.0 ** -23 + 2.0 ** -24 + (blocks + 8) * 2.0 ** -24)
            if cut:
                mag = mag + 7 * 2.0 ** -13 * (largest(x[:, at]) @ largest(w[:, at]).T) * np.abs(f)
        bound = mag
        if bias is not None:
            y = y + np.asarray(bias, np.float64)
            bound = bound + 2.0 ** -24 * (np.abs(y) + bound)
    return y, bound


def sort(ids, experts):
    """(offsets, tokens, slots) of ids [T, k], pair by pair."""
    ids = np.asarray(ids)
    t, k = ids.shape
    places = [[] for _ in range(experts)]
    for p, e in enumerate(ids.reshape(-1).tolist()):
        if 0 <= e < experts:
            places[e].append(p)
    order = [p for place in places for p in place]
    offsets = np.cumsum([0] + [len(p) for p in places]).astype(np.int32)
    tokens, slots = np.full(t * k, -1, np.int32), np.full(t * k, -1, np.int32)
    for s, p in enumerate(order):
        tokens[s], slots[p] = p // k, s
    return offsets, tokens, slots.reshape(t, k)


def combine(y, slots, w=None):
    """(out, bound) in fp64: each token's weighted sum and its fp32 evaluation's distance (an fma per row)."""
    y, out = np.asarray(y, np.float64), []
    rows = y[np.clip(slots, 0, max(len(y) - 1, 0))] if len(y) else np.zeros((*slots.shape, y.shape[1]))
    has = ((slots >= 0) & (slots < len(y)))[..., None]
    terms = np.where(has, rows, 0.0) * (1.0 if w is None else np.asarray(w, np.float64)[..., None])
    out = terms.sum(1)
    return out, np.abs(terms).sum(1) * slots.shape[1] * 2.0 ** -24


def combine_grad(dout, y, slots, w):
    """(dy, dw, bound of dw) in fp64.  A dot of H products: an fma each in fp32, in any order."""
    dout, y, w = np.asarray(dout, np.float64), np.asarray(y, np.float64), np.asarray(w, np.float64)
    dy, dw, bound = np.zeros_like(y), np.zeros(slots.shape), np.zeros(slots.shape)
    for t, j in zip(*np.nonzero((slots >= 0) & (slots < len(y)))):
        dy[slots[t, j]] = w[t, j] * dout[t]
        dw[t, j] = dout[t] @ y[slots[t, j]]
        bound[t, j] = np.abs(dout[t]) @ np.abs(y[slots[t, j]]) * (y.shape[1] + 16) * 2.0 ** -24
    return dy, dw, bound
