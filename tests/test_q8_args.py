"""The 8-bit activation path without a GPU: argument errors are found before
any launch, and the oracle agrees with torch's own expressions."""
import numpy as np
import pytest
import torch

from oracle import formats as fm
from oracle import q8 as o8


@pytest.fixture(scope="module")
def L():
    import _fp4x
    return _fp4x


P = 1 << 20      # an address that is aligned to everything and never read


def norm(L, x=P, xs=64, dt=0, r=None, rs=0, rdt=0, w=P, wdt=0, eps=1e-6, M=2, H=64, fmt=0, q=P, qs=64, s=P, ho=None,
         hs=0, y=None, ys=0):
    return L.lib().fp4x_rms_norm_q8(x, xs, dt, r, rs, rdt, w, wdt, 0.0, eps, M, H, fmt, q, qs, s, ho, hs, y, ys, None)


def test_norm_refusals(L):
    for kw in (dict(dt=3), dict(M=-1), dict(H=0), dict(H=32769), dict(fmt=3), dict(fmt=-1), dict(fmt=2, H=40),
               dict(x=None), dict(q=None), dict(s=None), dict(w=None), dict(x=P + 1), dict(s=P + 2), dict(xs=-64),
               dict(qs=63), dict(rdt=2), dict(wdt=2), dict(eps=-1e-6), dict(eps=float("nan")), dict(w=P + 1),
               dict(r=P + 1, rs=64), dict(r=P, rs=64, rdt=1, ho=P + 2, hs=64), dict(ho=P, hs=64),
               dict(r=P, rs=64, ho=P, hs=63), dict(r=P, rs=-64), dict(y=P, ys=63), dict(y=P + 1, ys=64)):
        assert norm(L, **kw) == L.ERR_ARG, kw
        assert L.lib().fp4x_last_error().startswith(b"rms_norm_q8")
    assert norm(L, M=0) == L.OK                       # no rows: nothing to launch
    assert norm(L, M=0, x=None, q=None, s=None, w=None) == L.OK


def test_silu_and_quantize_refusals(L):
    lib = L.lib()
    assert lib.fp4x_silu_mul_q8(P, 64, None, 64, 0, 2, 64, 0, P, 64, P, None) == L.ERR_ARG
    assert lib.fp4x_silu_mul_q8(P, 64, P + 1, 64, 0, 2, 64, 0, P, 64, P, None) == L.ERR_ARG
    assert lib.fp4x_silu_mul_q8(P, 64, P, -1, 0, 2, 64, 0, P, 64, P, None) == L.ERR_ARG
    assert lib.fp4x_silu_mul_q8(P, 64, P, 64, 0, 2, 65, 2, P, 65, P, None) == L.ERR_ARG
    assert lib.fp4x_silu_mul_q8(P, 64, P, 64, 0, 0, 64, 0, P, 64, P, None) == L.OK
    assert lib.fp4x_quantize_q8(P, 64, 1, 2, 64, 0, P, 32, P, None) == L.ERR_ARG
    assert lib.fp4x_quantize_q8(P + 2, 64, 1, 2, 64, 0, P, 64, P, None) == L.ERR_ARG
    assert lib.fp4x_quantize_q8(P, 64, 1, 0, 64, 0, P, 64, P, None) == L.OK


def linear(L, x=P, xs=64, sx=P, w=P, ws=64, sw=P, b=None, o=P, os=48, dt=0, M=2, N=48, K=64):
    return L.lib().fp4x_w8a8_linear(x, xs, sx, w, ws, sw, b, o, os, dt, M, N, K, None)


def test_linear_refusals(L):
    for kw in (dict(M=-1), dict(N=0), dict(K=0), dict(K=131072, xs=131072, ws=131072), dict(dt=3), dict(x=None),
               dict(sx=None), dict(w=None), dict(sw=None), dict(o=None), dict(x=P + 8), dict(w=P + 8), dict(xs=72),
               dict(ws=72), dict(xs=48), dict(ws=48), dict(sx=P + 2), dict(sw=P + 2), dict(b=P + 2), dict(o=P + 1),
               dict(o=P + 2, dt=1), dict(os=47), dict(M=(1 << 24) + 1), dict(N=(1 << 24) + 1),
               dict(M=1 << 20, N=1 << 18, os=1 << 18), dict(xs=1 << 24), dict(ws=1 << 24)):
        assert linear(L, **kw) == L.ERR_ARG, kw
        assert L.lib().fp4x_last_error().startswith(b"w8a8_linear")
    assert linear(L, M=0) == L.OK


def test_cpu_tensors_raise():
    import fp4x_kernels as F
    x, w = torch.ones((2, 64)).bfloat16(), torch.ones(64).bfloat16()
    q = torch.ones((2, 64), dtype=torch.int8)
    for call in (lambda: F.rms_norm_q8(x, w), lambda: F.silu_mul_q8(x), lambda: F.quantize_q8(x),
                 lambda: F.w8a8_linear(q, torch.ones(2), q, torch.ones(2))):
        with pytest.raises(RuntimeError):
            call()


def test_wrong_types_raise():
    import _fp4x
    import fp4x_kernels as F
    x = torch.ones((2, 64)).bfloat16()
    for call in (lambda: F.quantize_q8("x"), lambda: F.quantize_q8(None), lambda: F.silu_mul_q8([1.0]),
                 lambda: F.rms_norm_q8(x, None), lambda: F.w8a8_linear(x, x, x, 3)):
        with pytest.raises(TypeError):
            call()
    for name, n in (("rms_norm_q8", 8), ("silu_mul_q8", 3), ("quantize_q8", 2), ("w8a8_linear", 6)):
        with pytest.raises(TypeError):
            getattr(_fp4x.host(), name)(*[x] * (n - 1))


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "mx8"])
def test_oracle_against_torch(fmt):
    """The oracle's codes are the nearest ones: no other code of the format is closer to v / s."""
    rng = np.random.default_rng(3)
    v = (rng.standard_normal((6, 64)) * np.exp(rng.standard_normal((6, 1)))).astype(np.float32)
    q, s = o8.quantize(v, fmt)
    sv = np.repeat(np.exp2(s.astype(np.float64) - 127), 32, -1) if fmt == "mx8" else s.astype(np.float64)[:, None]
    grid = np.arange(-127, 128) if fmt == "int8" else np.sort(fm.e4m3_decode(
        np.array([c for c in range(256) if c & 127 != 127], np.uint8)))
    got = q.astype(np.float64) if fmt == "int8" else fm.e4m3_decode(q).astype(np.float64)
    y = v / sv
    assert (np.abs(got - y) <= np.abs(y[..., None] - grid).min(-1) + 1e-6 * np.abs(y)).all()
    t = torch.from_numpy(v)
    if fmt == "int8":
        ts = t.abs().amax(-1) / 127
        assert np.array_equal(s, ts.numpy()) and np.array_equal(q, torch.round(t / ts[:, None]).to(torch.int8).numpy())
    if fmt == "mx8":
        import fp4x_kernels as F
        tq, te = F.quantize_mx8(t)
        assert np.array_equal(q, tq.numpy()) and np.array_equal(s, te.numpy())


def test_oracle_norm_against_fp64():
    rng = np.random.default_rng(4)
    x, r, w = (rng.standard_normal(s).astype(np.float32) for s in ((5, 200), (5, 200), (200,)))
    v, h = o8.rms_norm(x, w, 1e-6, r, lambda a: a)
    d = x.astype(np.float64) + r
    assert (np.abs(h - d) <= 2.0 ** -24 * np.abs(d)).all()
    want = h * w.astype(np.float64) / np.sqrt((h.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-6)
    assert (np.abs(v - want) <= 3.01 * 2.0 ** -24 * np.abs(want)).all()      # rs, h * rs and the product by w


def test_oracle_product():
    rng = np.random.default_rng(5)
    x, w = rng.integers(-128, 128, (4, 999)).astype(np.int8), rng.integers(-128, 128, (7, 999)).astype(np.int8)
    one = np.ones(7, np.float32)
    want = x.astype(np.int64) @ w.astype(np.int64).T
    assert np.array_equal(o8.w8a8(x, one[:4], w, one), want.astype(np.float32))
