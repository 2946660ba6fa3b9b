"""e4m3 in blocks of 128 and experts without a GPU: argument errors are found
before any launch, and the oracle agrees with torch's own expressions."""
import numpy as np
import pytest
import torch

from oracle import f8 as o
from oracle import formats as fm


@pytest.fixture(scope="module")
def L():
    import _fp4x
    return _fp4x


P = 1 << 20      # an address that is aligned to everything and never read


def refused(L, rc, who):
    return rc == L.ERR_ARG and L.lib().fp4x_last_error().startswith(who)


def linear(L, x=P, xs=64, sx=P, sr=1, sb=2, w=P, ws=64, sw=P, b=None, out=P, os=48, dt=0, M=2, N=48, K=64):
    return L.lib().fp4x_f8_linear(x, xs, sx, sr, sb, w, ws, sw, b, out, os, dt, M, N, K, None)


COMMON = (dict(M=-1), dict(N=0), dict(K=0), dict(K=131072, xs=131072, ws=131072), dict(dt=3), dict(x=None), dict(sx=None), dict(w=None),
          dict(sw=None), dict(out=None), dict(x=P + 8), dict(w=P + 8), dict(xs=72), dict(ws=72), dict(xs=48), dict(ws=48), dict(sx=P + 2),
          dict(sw=P + 2), dict(out=P + 1), dict(out=P + 2, dt=1), dict(os=47), dict(N=(1 << 24) + 1), dict(xs=1 << 24), dict(ws=1 << 24),
          dict(sr=-1), dict(sb=-1), dict(sr=1 << 22))


def test_linear_refusals(L):
    for kw in COMMON + (dict(b=P + 2), dict(M=(1 << 24) + 1), dict(M=1 << 20, N=1 << 18, os=1 << 18), dict(M=1 << 14, N=1 << 23, os=1 << 23, dt=1, K=16)):
        assert refused(L, linear(L, **kw), b"f8_linear:"), kw
    assert linear(L, M=0) == L.OK and linear(L, M=0, x=None, out=None) == L.OK


def experts(L, x=P, xs=64, sx=P, sr=1, sb=2, X=2, tok=None, off=P, E=3, w=P, ws=64, we=64 * 48, sw=P, out=P, os=48, dt=0, M=2, N=48, K=64):
    return L.lib().fp4x_f8_linear_experts(x, xs, sx, sr, sb, X, tok, off, E, w, ws, we, sw, out, os, dt, M, N, K, None)


def test_experts_refusals(L):
    for kw in COMMON + (dict(E=0), dict(E=4097), dict(off=None), dict(off=P + 2), dict(tok=P + 2), dict(we=-64), dict(we=72), dict(X=1),
                        dict(tok=P, X=0), dict(tok=P, X=1 << 26), dict(tok=P, X=1 << 12, sr=1 << 21), dict(M=(1 << 24) + 1, X=1 << 25)):
        assert refused(L, experts(L, **kw), b"f8_linear_experts:"), kw
    assert experts(L, M=0) == L.OK and experts(L, M=0, off=None) == L.OK


def test_forms(L):
    assert L.lib().fp4x_f8_form(0, 1, 1, 0) == -1 and L.lib().fp4x_f8_experts_form(1, 1, 1, 0, 0) == -1


def test_quantize_refusals(L):
    lib = L.lib()

    def q(w=P, wr=64, we=64 * 8, dt=0, E=2, N=8, K=64, c=P, cr=64, ce=64 * 8, s=P):
        return lib.fp4x_quantize_f8(w, wr, we, dt, E, N, K, c, cr, ce, s, None)
    for kw in (dict(dt=3), dict(E=-1), dict(N=-1), dict(K=0), dict(K=(1 << 24) + 1), dict(w=None), dict(c=None), dict(s=None), dict(w=P + 1),
               dict(s=P + 2), dict(wr=-1), dict(we=-1), dict(cr=63), dict(ce=500)):
        assert refused(L, q(**kw), b"quantize_f8"), kw
    assert q(N=0) == L.OK and q(E=0, w=None) == L.OK
    for fmt in (3, 5):                               # 4 is e4m3_g128
        assert lib.fp4x_quantize_q8(P, 64, 0, 2, 64, fmt, P, 64, P, None) == L.ERR_ARG
    assert lib.fp4x_quantize_q8(P, 64, 0, 2, 64, 4, P, 64, P + 2, None) == L.ERR_ARG
    assert lib.fp4x_quantize_q8(P, 64, 0, 0, 64, 4, P, 64, P, None) == L.OK


def test_sort_refusals(L):
    lib = L.lib()

    def sort(ids=P, wide=1, row=8, T=3, k=8, E=64, off=P, tok=P, slots=P, ws=None, n=0):
        return lib.fp4x_expert_sort(ids, wide, row, T, k, E, off, tok, slots, ws, n, None)
    for kw in (dict(T=-1), dict(k=0), dict(k=(1 << 20) + 1), dict(E=0), dict(E=4097), dict(T=(1 << 27) + 1), dict(off=None), dict(off=P + 2),
               dict(ids=None), dict(ids=P + 4), dict(ids=P + 2, wide=0), dict(tok=None), dict(slots=None), dict(tok=P + 1), dict(slots=P + 2),
               dict(row=-1), dict(T=4000), dict(T=4000, ws=P, n=100), dict(T=4000, ws=P + 2, n=1 << 20)):
        assert refused(L, sort(**kw), b"expert_sort"), kw


def test_rows_and_combine_refusals(L):
    lib = L.lib()

    def rows(x=P, xs=64, el=2, T=3, tok=P, M=5, H=64, out=P, os=64):
        return lib.fp4x_expert_rows(x, xs, el, T, tok, M, H, out, os, None)
    for kw in (dict(T=-1), dict(M=-1), dict(H=0), dict(el=3), dict(el=8), dict(x=None), dict(tok=None), dict(out=None), dict(tok=P + 2),
               dict(xs=-1), dict(os=63)):
        assert refused(L, rows(**kw), b"expert_rows"), kw
    assert rows(M=0, tok=None, out=None) == L.OK

    def combine(y=P, ys=64, dt=0, M=24, slots=P, w=P, wdt=1, out=P, os=64, T=3, k=8, H=64):
        return lib.fp4x_expert_combine(y, ys, dt, M, slots, w, wdt, out, os, T, k, H, None)
    for kw in (dict(dt=3), dict(wdt=3), dict(T=-1), dict(k=0), dict(M=-1), dict(H=0), dict(y=None), dict(slots=None), dict(out=None),
               dict(slots=P + 2), dict(y=P + 1), dict(out=P + 1), dict(w=P + 2), dict(ys=-1), dict(os=63)):
        assert refused(L, combine(**kw), b"expert_combine:"), kw
    assert combine(T=0, slots=None) == L.OK

    def grad(d=P, ds=64, y=P, ys=64, dt=0, M=24, slots=P, tok=P, w=P, wdt=1, dy=P, dys=64, dw=P, T=3, k=8, H=64):
        return lib.fp4x_expert_combine_grad(d, ds, y, ys, dt, M, slots, tok, w, wdt, dy, dys, dw, T, k, H, None)
    for kw in (dict(dt=3), dict(wdt=3), dict(T=-1), dict(k=0), dict(k=129), dict(M=-1), dict(H=0), dict(H=32769), dict(d=None), dict(y=None),
               dict(slots=None), dict(tok=None), dict(w=None), dict(dy=None), dict(dw=None), dict(tok=P + 2), dict(slots=P + 1), dict(d=P + 1),
               dict(dy=P + 1), dict(w=P + 2), dict(dw=P + 2), dict(ds=-1), dict(ys=-1), dict(dys=63)):
        assert refused(L, grad(**kw), b"expert_combine_grad"), kw
    assert refused(L, grad(T=1 << 26, k=1, dys=64), b"expert_combine_grad: tokens times")
    assert grad(T=0, M=0, d=None, y=None, dy=None) == L.OK


# ------------------------------------------------------------------ the oracle
def test_oracle_codes():
    rng = np.random.default_rng(0)
    v = (rng.standard_normal((9, 300)) * np.exp(3 * rng.standard_normal((9, 1)))).astype(np.float32)
    q, s = o.quantize_rows(v)
    t = torch.from_numpy(v)
    for b in range(3):
        at = slice(128 * b, 128 * b + 128)
        amax = t[:, at].abs().amax(1, keepdim=True)
        st = amax / torch.full_like(amax, 448.0)
        assert np.array_equal(s[:, b], st[:, 0].numpy())
        assert np.array_equal(q[:, at], (t[:, at] / st).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    w = v.reshape(270, 10).T.copy()                  # [10, 270]
    q, s = o.quantize_weight(w)
    assert s.shape == (1, 3) and s[0, 2] == np.abs(w[:, 256:]).max() / np.float32(448)
    assert np.array_equal(q, o.quantize_weight(np.vstack([w, 0 * w]))[0][:10])


def test_oracle_product_and_its_bound():
    rng = np.random.default_rng(1)
    (xq, xs), (wq, ws) = o.quantize_rows(rng.standard_normal((5, 300)).astype(np.float32)), o.quantize_weight(rng.standard_normal((130, 300)).astype(np.float32))
    y, bound = o.linear(xq, xs, wq, ws)
    x = fm.e4m3_decode(xq).astype(np.float64) * np.repeat(xs, 128, 1)[:, :300]
    w = fm.e4m3_decode(wq).astype(np.float64) * np.repeat(np.repeat(ws, 128, 0)[:130], 128, 1)[:, :300]
    assert np.allclose(y, x @ w.T, rtol=1e-12, atol=1e-12)
    # fp32 products added one by one in fp32 stay within the bound
    got = np.zeros((5, 130), np.float32)
    cut = np.zeros((5, 130))
    for b in range(3):
        at = slice(128 * b, 128 * b + 128)
        p = fm.e4m3_decode(xq[:, at]).astype(np.float32)[:, None] * fm.e4m3_decode(wq[:, at]).astype(np.float32)[None]
        f = xs[:, b:b + 1] * np.repeat(ws[:, b], 128)[None, :130]
        part = np.zeros((5, 130), np.float32)
        for i in range(p.shape[2]):
            part = part + p[:, :, i]
        got = got + part * f
        # and the fp8 instruction's: eight at a time, each cut to 2^-13 of the power of two of the largest
        for i in range(0, p.shape[2], 8):
            e = np.abs(p[:, :, i:i + 8]).astype(np.float64)
            top = np.exp2(np.floor(np.log2(np.maximum(e.max(-1, keepdims=True), 2.0 ** -18))) - 13)
            cut += (np.sign(p[:, :, i:i + 8]) * np.floor(e / top) * top).sum(-1) * f
    assert (np.abs(got - y) <= bound).all() and np.abs(got - y).max() > 0
    loose = o.linear(xq, xs, wq, ws, cut=True)[1]
    assert (np.abs(cut - y) <= loose).all() and (loose > bound).all() and np.abs(cut - y).max() > np.abs(got - y).max()


def test_oracle_sort():
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(-1, 9, (40, 3), generator=g)
    offsets, tokens, slots = o.sort(ids.numpy(), 8)
    flat = torch.where((ids < 0) | (ids >= 8), 8, ids).reshape(-1)
    key, order = torch.sort(flat, stable=True)
    n = int((key < 8).sum())
    assert offsets[8] == n and np.array_equal(offsets, np.searchsorted(key.numpy(), np.arange(9)))
    assert np.array_equal(tokens[:n], (order // 3).numpy()[:n]) and (tokens[n:] == -1).all()
    assert all(slots.reshape(-1)[order[i]] == i for i in range(n)) and (slots.reshape(-1)[order[n:].numpy()] == -1).all()


def test_oracle_combine_and_gradient():
    """The sum and its gradients against torch's own differentiation in fp64."""
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(-1, 6, (20, 4), generator=g)
    _, tokens, slots = o.sort(ids.numpy(), 6)
    y = torch.randn((80, 7), generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.rand((20, 4), generator=g, dtype=torch.float64, requires_grad=True)
    d = torch.randn((20, 7), generator=g, dtype=torch.float64)
    s = torch.from_numpy(slots).long()
    out = torch.where((s < 0)[..., None], torch.zeros((), dtype=torch.float64), y[s.clamp_min(0)] * w[..., None]).sum(1)
    out.backward(d)
    got, bound = o.combine(y.detach().numpy(), slots, w.detach().numpy())
    assert np.allclose(got, out.detach().numpy()) and (bound >= 0).all()
    dy, dw, _ = o.combine_grad(d.numpy(), y.detach().numpy(), slots, w.detach().numpy())
    assert np.allclose(dy, y.grad.numpy()) and np.allclose(dw, w.grad.numpy())
    x = torch.randn((20, 7), generator=g, dtype=torch.float64, requires_grad=True)
    t = torch.from_numpy(tokens).long()
    rows = torch.where((t < 0)[:, None], torch.zeros((), dtype=torch.float64), x[t.clamp_min(0)])
    rows.backward(torch.from_numpy(dy))
    assert np.allclose(o.combine(dy, slots)[0], x.grad.numpy())
