"""Rows in 8 bits, their norm and the int8 product, restated in numpy (oracle;
test infrastructure only).

Every step is one rounded fp32 operation but the norm's mean square, which is
taken in fp64; numpy's fp32 arithmetic rounds each operation to nearest even,
so codes, scales and outputs are defined to the last bit.
"""
import numpy as np

from .formats import F32, e4m3_encode

MIN_AMAX = F32(1e-12)


def quantize(v, fmt):
    """(codes, scales) of fp32 rows v [M, H]: int8 codes and fp32 [M] ("int8"),
    e4m3fn codes (u8) and fp32 [M] ("e4m3"), e4m3fn codes (u8) and e8m0 (u8)
    [M, H/32] ("mx8").  Rows (blocks) with an infinity or a NaN: scale NaN
    (255), codes 0 (0x7f)."""
    v = np.asarray(v, F32)
    m, h = v.shape
    if fmt == "mx8":
        b = v.reshape(m, h // 32, 32)
        bad = ~np.isfinite(b).all(-1)
        b = np.where(bad[..., None], F32(0), b)
        e = (np.abs(b).max(-1).view(np.uint32) >> 23).astype(np.int64)
        X = np.where(e == 0, -127, np.maximum(e - 127 - 8, -127))
        y = (b.astype(np.float64) * np.exp2(-X.astype(np.float64))[..., None]).astype(F32)
        q = e4m3_encode(y, saturate=True)
        q = np.where(bad[..., None], 0x7f, q).astype(np.uint8)
        return q.reshape(m, h), np.where(bad, 255, X + 127).astype(np.uint8)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[:, None], F32(0), v)
    s = np.maximum(np.abs(v).max(-1), MIN_AMAX) / F32(127 if fmt == "int8" else 448)
    y = v / s[:, None]
    q = np.rint(y).astype(np.int8) if fmt == "int8" else e4m3_encode(y, saturate=True).astype(np.uint8)
    return q, np.where(bad, F32(np.nan), s)


def rms_norm(x, w, eps, res=None, round_res=None, w_offset=0.0):
    """(v, h) in fp32: h = round_res(x + res) or x, v = (h * rs) * (w + w_offset)."""
    h = np.asarray(x, F32)
    with np.errstate(all="ignore"):
        if res is not None:
            h = round_res(h + np.asarray(res, F32))
        d = h.astype(np.float64)
        rs = (1.0 / np.sqrt((d * d).sum(-1, keepdims=True) / h.shape[1] + float(eps))).astype(F32)
        return (h * rs) * (np.asarray(w, F32) + F32(w_offset)), h


def silu_mul(g, u):
    """silu(g) * u in fp64."""
    g, u = np.asarray(g, np.float64), np.asarray(u, np.float64)
    with np.errstate(all="ignore"):
        return g / (1.0 + np.exp(-g)) * u


def w8a8(xq, xs, wq, ws, bias=None):
    """fp32 [M, N] before the output cast: ((fp32(sum) * xs) * ws) + bias, the
    sum in int64 (here through fp64, which holds it exactly)."""
    acc = (xq.astype(np.float64) @ wq.astype(np.float64).T).astype(F32)
    with np.errstate(all="ignore"):
        y = (acc * np.asarray(xs, F32)[:, None]) * np.asarray(ws, F32)
        return y if bias is None else y + np.asarray(bias, F32)
