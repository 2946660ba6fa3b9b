"""The 8-bit activation path on the GPU (csrc/fp4x_rowq.hip, csrc/fp4x_i8.hip):
norms, rows and products equal the oracle bit for bit (every step is one
rounded fp32 operation on exact sums); the gated activation is within the
roundings of its fp32 evaluation."""
import numpy as np
import pytest
import torch

from oracle import formats as fm
from oracle import q8 as o8

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def F(gpu):
    import fp4x_kernels
    return fp4x_kernels


def host(t):
    """Values of a float tensor as fp32, codes and scales as they are."""
    if t.dtype in (torch.bfloat16, torch.float16):
        return t.float().cpu().numpy()
    if t.dtype == torch.float8_e4m3fn:
        return t.view(torch.uint8).cpu().numpy()
    return t.cpu().numpy()


def rounder(dt):
    def r(a):
        with np.errstate(all="ignore"):
            return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(DT[dt]).float().numpy()
    return r


def same(got, want, what):
    got, want = np.ascontiguousarray(host(got)), np.ascontiguousarray(want)
    assert got.shape == want.shape, what
    if want.dtype.kind == "f":
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got), nan), what
        got, want = np.where(nan, 0, got), np.where(nan, 0, want)
        bad = got.view(np.uint32) != want.astype(np.float32).view(np.uint32)
        bad &= ~((got == 0) & (want == 0))           # the sign of a zero is not held to
    else:
        bad = got != want
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist())


def rows(seed, m, h, dt, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, h), generator=g) * scale * torch.exp(torch.randn((m, 1), generator=g))
    return x.to(DT[dt])


def check_norm(F, x, w, r=None, fmt="int8", eps=1e-6, off=0.0, normed=True, rdt=None, xdt="bf16"):
    """x, w, r: CPU tensors (any strides), moved to the GPU with their layout."""
    def up(t):
        if t is None:
            return None
        base = torch.empty(0, dtype=t.dtype).set_(t.untyped_storage()) if t.storage_offset() or not t.is_contiguous() else t
        return base.cuda().as_strided(t.shape, t.stride(), t.storage_offset()) if base is not t else t.cuda()
    got = F.rms_norm_q8(up(x), up(w), eps=eps, residual=up(r), fmt=fmt, w_offset=off, normed=normed)
    v, h = o8.rms_norm(x.float().numpy(), w.float().numpy(), eps, None if r is None else r.float().numpy(),
                       rounder(rdt or xdt), off)
    q, s = o8.quantize(v, fmt)
    want = [(q, "codes"), (s, "scales")] + ([(h, "residual")] if r is not None else [])
    want += [(rounder(xdt)(v), "normed")] if normed else []
    assert len(got) == len(want)
    for g, (t, what) in zip(got, want):
        same(g, t, what)


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "mx8"])
@pytest.mark.parametrize("xdt,rdt,wdt", [("bf16", None, "bf16"), ("bf16", "bf16", "bf16"), ("bf16", "f32", "f32"),
                                         ("f16", "f16", "f32"), ("f16", "f32", "f16"), ("bf16", "bf16", "f32"),
                                         ("f16", "f16", "f16"), ("f32", "f32", "f32")])
def test_norm_types(F, fmt, xdt, rdt, wdt):
    for seed, (m, h) in enumerate([(3, 2560), (5, 96), (2, 12288)]):
        x, w = rows(seed, m, h, xdt), (1 + 0.3 * rows(50 + seed, 1, h, "f32")[0]).to(DT[wdt])
        r = None if rdt is None else rows(90 + seed, m, h, rdt, 3.0)
        check_norm(F, x, w, r, fmt, off=0.25 * seed, rdt=rdt, xdt=xdt)


# every lane count per row (4 .. 1024), chunks per lane (1, 2, 4), rows that end inside a chunk, several rows per wave
@pytest.mark.parametrize("h", [1, 2, 7, 8, 9, 15, 31, 33, 64, 65, 127, 129, 255, 257, 511, 520, 1025, 2571, 4097, 8191,
                               8193, 8200, 16384, 16385, 20001, 32768])
def test_norm_lengths(F, h):
    for m in (1, 9):
        x, w = rows(h, m, h, "bf16"), (1 + 0.3 * rows(h + 1, 1, h, "f32")[0]).bfloat16()
        check_norm(F, x, w, rows(h + 2, m, h, "bf16"), "int8", rdt="bf16")
        check_norm(F, x.half(), w.half(), None, "e4m3", xdt="f16")


def test_norm_many_rows(F):
    x, w = rows(1, 70001, 40, "bf16"), (1 + 0.3 * rows(2, 1, 40, "f32")[0]).bfloat16()
    check_norm(F, x, w, rows(3, 70001, 40, "bf16"), "int8", rdt="bf16")
    # more rows than the grid has workgroups (2^20, one row of four lanes each is 64 rows a workgroup: a row of 600 is one)
    x = torch.full(((1 << 20) + 3, 600), 1.0, dtype=torch.bfloat16, device="cuda")
    x[-1] = 2.0
    q, s = F.quantize_q8(x)
    assert bool((q == 127).all()) and float(s[-1]) == np.float32(2.0) / np.float32(127)
    assert bool((s[:-1] == float(np.float32(1.0) / np.float32(127))).all())


# 2, 3 and 4 chunks of 8 per lane: with few rows only rows past 8192 values take those
MANY = [(2100, 520), (1500, 1025), (700, 2571), (430, 6144), (400, 6145), (300, 8191), (280, 12000), (130, 32766)]


@pytest.mark.parametrize("m,h", MANY)
def test_many_rows(F, m, h):
    r = rows(h + 2, m, h, "f32")
    for xdt, rdt, fmt in (("bf16", "bf16", "int8"), ("f16", "f32", "e4m3"), ("f32", "f32", "int8")):
        x, w = rows(h, m, h, xdt), (1 + 0.3 * rows(h + 1, 1, h, "f32")[0]).to(DT[xdt])
        check_norm(F, x, w, r.to(DT[rdt]), fmt, rdt=rdt, xdt=xdt)
        q, s = F.quantize_q8(x.cuda(), fmt)
        a, b = codes_of(x, fmt)
        same(q, a, "codes")
        same(s, b, "scales")
        # the gate and the up rows change no row but their own, whatever the number of rows
        q, s = F.silu_mul_q8(x.cuda(), r.to(x.dtype).cuda(), fmt)
        for i in (0, m // 2, m - 1):
            q1, s1 = F.silu_mul_q8(x[i:i + 1].cuda(), r[i:i + 1].to(x.dtype).cuda(), fmt)
            same(q[i:i + 1], host(q1), i)
            same(s[i:i + 1], host(s1), i)
    if h % 32 == 0:
        x = rows(h, m, h, "bf16")
        check_norm(F, x, (1 + 0.3 * rows(h + 1, 1, h, "f32")[0]).bfloat16(), None, "mx8")


def test_norm_strides_and_alignment(F):
    base = rows(7, 6, 700, "bf16")
    w = (1 + 0.3 * rows(8, 1, 701, "f32")[0]).bfloat16()
    check_norm(F, base[:, 1:], w[1:700], base[:, :-1], "int8", rdt="bf16")          # rows off every alignment
    check_norm(F, base[::2, 3:300], w[:297], None, "e4m3")
    check_norm(F, base[1:2].expand(4, 700), w[:700], None, "int8")                   # one row read four times
    check_norm(F, base.t(), w[:6], None, "int8")                                     # another column stride: copied


def test_norm_residual_in_place(F):
    x, r, w = rows(1, 33, 2560, "bf16").cuda(), rows(2, 33, 2560, "bf16").cuda(), torch.ones(2560).bfloat16().cuda()
    q, s, h = F.rms_norm_q8(x, w, residual=r)
    r2 = r.clone()
    q2, s2, h2 = F.rms_norm_q8(x, w, residual=r2, residual_out=r2)
    assert h2.data_ptr() == r2.data_ptr()
    assert torch.equal(h, r2) and torch.equal(q, q2) and torch.equal(s, s2)
    for hh in (17, 2571, 9001):                     # rows whose last chunk overlaps the one before
        x, r, w = rows(3, 5, hh, "bf16").cuda(), rows(4, 5, hh, "bf16").cuda(), torch.ones(hh).bfloat16().cuda()
        want = F.rms_norm_q8(x, w, residual=r)
        got = F.rms_norm_q8(x, w, residual=r, residual_out=r)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_norm_degenerate_rows(F):
    h = 96
    x = rows(5, 10, h, "f32")
    x[0] = 0
    x[1, 17] = float("inf")
    x[2, 40] = float("nan")
    x[3, 95] = float("-inf")
    x[4] = 1e-30
    x[5] = 1e30
    x[6, :] = 0
    x[6, 5] = 3e38
    x[7] = 1e-42                                     # fp32 subnormals
    w = torch.ones(h)
    for fmt in ("int8", "e4m3", "mx8"):
        check_norm(F, x, w, None, fmt, xdt="f32")
        check_norm(F, x, w, x.flip(0), fmt, eps=0.0 if fmt == "int8" else 1e-6, xdt="f32", rdt="f32")


def codes_of(x, fmt):
    return o8.quantize(x.float().numpy(), fmt)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "mx8"])
def test_quantize(F, fmt, dt):
    for seed, (m, h) in enumerate([(1, 32), (7, 2560), (300, 640), (3, 16384), (2, 32768)]):
        x = rows(seed, m, h, dt)
        q, s = F.quantize_q8(x.cuda(), fmt)
        a, b = codes_of(x, fmt)
        same(q, a, "codes")
        same(s, b, "scales")


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "mx8"])
def test_quantize_every_bf16(F, fmt):
    """Every bf16 value, infinities and NaN among them, beside ordinary ones; ties and the formats' subnormals."""
    bits = np.arange(65536, dtype=np.uint16).reshape(1024, 64)
    rng = np.random.default_rng(0)
    bits = rng.permutation(bits.reshape(-1)).reshape(1024, 64)
    x = torch.from_numpy(fm.bf16_to_f32(bits)).bfloat16()
    x = torch.cat([x, x.float().clamp(-4, 4).nan_to_num(1.0).bfloat16()])
    q, s = F.quantize_q8(x.cuda(), fmt)
    a, b = codes_of(x, fmt)
    same(q, a, "codes")
    same(s, b, "scales")
    ties = torch.arange(-127, 128).repeat(2, 1).float() / 2    # amax 63.5: quotients on halves
    ties = torch.nn.functional.pad(ties, (0, 1), value=127.0)
    q, s = F.quantize_q8(ties.cuda(), fmt)
    a, b = codes_of(ties, fmt)
    same(q, a, "ties")


def test_quantize_odd_rows_lie_on_16_bytes(F):
    for k in (1, 5, 15, 17, 2571):
        x = rows(k, 4, k, "bf16")
        q, s = F.quantize_q8(x.cuda())
        assert q.shape == (4, k) and q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
        same(q, codes_of(x, "int8")[0], k)


# silu(g) * u in fp32: expf within 1 ulp (2^-23 relative), 1 + t, two products (2^-24 each) and v_rcp_f32 within 1 ulp,
# so v is within 7 steps of 2^-24; the scale adds its division and v's maximum: 8; the quotient 16 in all.
STEP = 2.0 ** -24


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "mx8"])
def test_silu_mul(F, fmt, dt):
    for seed, (m, f) in enumerate([(1, 32), (3, 640), (130, 6144), (5, 96)]):
        gu = rows(seed, m, 2 * f, dt, 2.0)
        q, s = F.silu_mul_q8(gu.cuda(), fmt=fmt)
        q2, s2 = F.silu_mul_q8(gu[:, :f].cuda(), gu[:, f:].cuda(), fmt=fmt)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
        v = o8.silu_mul(gu[:, :f].float().numpy(), gu[:, f:].float().numpy())
        if fmt == "mx8":
            _, e = o8.quantize(v.astype(np.float32), fmt)
            b = np.abs(v).reshape(m, -1, 32).max(-1)
            edge = np.abs(b / np.exp2(np.rint(np.log2(b))) - 1) < 8 * STEP      # a maximum beside a power of two
            se = host(s)
            assert (se[~edge] == e[~edge]).all() and (np.abs(se.astype(int) - e) <= 1).all()
            sv = np.repeat(np.exp2(se.astype(np.float64) - 127), 32, -1).reshape(m, f)
        else:
            top = 127 if fmt == "int8" else 448
            s64 = np.abs(v).max(-1) / top
            assert (np.abs(host(s) - s64) <= 8 * STEP * s64).all()
            sv = host(s).astype(np.float64)[:, None]
        y = v / sv
        got = host(q).astype(np.float64) if fmt == "int8" else fm.e4m3_decode(host(q)).astype(np.float64)
        half = 0.5 if fmt == "int8" else np.maximum(np.abs(y) * 2.0 ** -4, 2.0 ** -10)
        y = np.clip(y, -448, 448) if fmt == "mx8" else y
        assert (np.abs(got - y) <= half + 16 * STEP * np.abs(y)).all()


def test_silu_extremes(F):
    g = torch.tensor([[-200.0, -90.0, -87.0, -20.0, -1e-30, 0.0, 1e-30, 20.0, 90.0, 200.0] + [1.0] * 6])
    u = torch.full_like(g, 3.0)
    q, s = F.silu_mul_q8(g.cuda(), u.cuda(), fmt="e4m3")
    v = o8.silu_mul(g.numpy(), u.numpy())
    assert abs(float(s) - 600.0 / 448) <= 8 * STEP * 600 / 448
    d = fm.e4m3_decode(host(q)) * float(s)
    assert (np.abs(d - v) <= np.maximum(np.abs(v) * (2.0 ** -4 + 16 * STEP), float(s) * 2.0 ** -10)).all()
    g[0, 3] = float("nan")
    q, s = F.silu_mul_q8(g.cuda(), u.cuda())
    assert bool(s.isnan().all()) and not bool(q.any())


# ------------------------------------------------------------------ products
def int_codes(seed, n, k, lo=-127):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, 128, (n, k), generator=g, dtype=torch.int8), 0.01 * (0.5 + torch.rand(n, generator=g))


def padded(q):
    """q in rows of a multiple of 16 bytes, with the worst values in the gaps."""
    n, k = q.shape
    c = torch.full((n, (k + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")
    c[:, :k] = q.cuda()
    return c[:, :k]


def check_linear(F, m, n, k, out="bf16", bias=False, lo=-127, seed=0):
    xq, xs = int_codes(seed, m, k, lo)
    wq, ws = int_codes(seed + 1, n, k, lo)
    b = torch.randn(n, generator=torch.Generator().manual_seed(seed + 2)) if bias else None
    y = F.w8a8_linear(padded(xq), xs.cuda(), padded(wq), ws.cuda(), None if b is None else b.cuda(), DT[out])
    assert y.shape == (m, n) and y.dtype == DT[out]
    want = o8.w8a8(xq.numpy(), xs.numpy(), wq.numpy(), ws.numpy(), None if b is None else b.numpy())
    same(y, rounder(out)(want), (m, n, k, out))


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 33, 48, 63, 64, 65, 100, 128, 129, 200, 256, 257, 300, 513])
def test_linear_rows(F, m):
    check_linear(F, m, 640, 2560, seed=m)
    check_linear(F, m, 333, 592, "f32", True, seed=m)


@pytest.mark.parametrize("k", [1, 3, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 272, 384, 400, 1000, 2571, 6145])
def test_linear_lengths(F, k):
    for m, n in ((1, 48), (16, 100), (40, 33), (70, 260), (300, 520)):
        check_linear(F, m, n, k, "f32", seed=k)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 15, 16, 17, 31, 32, 33, 63, 65, 127, 129, 255, 257, 1000, 2561])
def test_linear_columns(F, n):
    for m in (1, 16, 33, 64, 130, 260):
        check_linear(F, m, n, 320, "f16", n % 2 == 0, seed=n)


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,n,k", [(4, 16384, 640), (64, 2560, 6144), (250, 1999, 2560), (1024, 1024, 1024),
                                   (700, 3001, 1216), (96, 16, 10240), (2049, 64, 512)])
def test_linear_sizes(F, m, n, k, out):
    check_linear(F, m, n, k, out, True)


# every form, K below and inside a unit, several tiles per workgroup
FORMS = [(1, 640), (40, 1000), (16, 18000), (100, 1280), (64, 5200), (33, 9001), (96, 13000), (250, 13310), (256, 16384),
         (700, 3001), (512, 16500), (1100, 16390), (4100, 4400), (9000, 70), (33, 40000), (1000, 5000)]
FORM_KS = [100, 320, 1400, 2571]


@pytest.mark.parametrize("k", FORM_KS)
@pytest.mark.parametrize("m,n", FORMS)
def test_linear_forms(F, m, n, k):
    out, bias = ("bf16", "f16", "f32")[(m + k) % 3], m % 2 == 0
    xq, xs = int_codes(m + k, m, k)
    wq, ws = int_codes(m + k + 1, n, k)
    b = torch.randn(n, generator=torch.Generator().manual_seed(m)) if bias else None
    y = F.w8a8_linear(padded(xq), xs.cuda(), padded(wq), ws.cuda(), None if b is None else b.cuda(), DT[out])
    rows = np.unique(np.r_[:min(m, 40), np.linspace(0, m - 1, 60).astype(int), max(0, m - 40):m])   # of large ones
    want = o8.w8a8(xq.numpy()[rows], xs.numpy()[rows], wq.numpy(), ws.numpy(), None if b is None else b.numpy())
    same(y[torch.from_numpy(rows).cuda()], rounder(out)(want), (m, n, k, out))


# many tiles of as many k-tiles as a form has stages, one more and one less
@pytest.mark.parametrize("m,n", [(2851, 18470), (1100, 16390), (2000, 9000), (600, 20000), (4100, 6000), (70, 60000)])
@pytest.mark.parametrize("k", [199, 256, 300, 384, 400, 512, 520, 640])
def test_linear_short_sums_of_many_tiles(F, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + k)
    xq, wq = (torch.randint(-128, 128, (r, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]
              for r in (m, n))
    xs, ws, b = (0.5 + torch.rand(r, generator=g, device="cuda") for r in (m, n, n))
    want = ((xq.float() @ wq.float().t()) * xs[:, None]) * ws + b   # sums below 2^24 are exact in fp32
    for _ in range(3):
        assert torch.equal(F.w8a8_linear(xq, xs, wq, ws, b, torch.float32), want)


def test_linear_forms_are_all_reached(F):
    import _fp4x
    form = _fp4x.lib().fp4x_w8a8_form
    assert {form(m, n, k) for m, n in FORMS for k in FORM_KS} == set(range(11))
    assert form(0, 1, 1) == form(1, 0, 1) == form(1, 1, 0) == -1


def test_linear_far_rows(F):
    """Strides up to the limit, and beyond it (copied)."""
    xq, xs = int_codes(1, 300, 200)
    wq, ws = int_codes(2, 50, 200)
    want = rounder("bf16")(o8.w8a8(xq.numpy(), xs.numpy(), wq.numpy(), ws.numpy()))
    for ld in ((1 << 24) - 16, 1 << 24):
        big = torch.empty(299 * ld + 208, dtype=torch.int8, device="cuda")
        x = big.as_strided((300, 200), (ld, 1))
        x.copy_(xq)
        same(F.w8a8_linear(x, xs.cuda(), wq.cuda(), ws.cuda()), want, ld)
        same(F.w8a8_linear(wq.cuda(), ws.cuda(), x, xs.cuda(), out_dtype=torch.float32),
             o8.w8a8(wq.numpy(), ws.numpy(), xq.numpy(), xs.numpy()), ld)


def test_linear_far_rows_of_a_large_tile(F):
    """Rows of one tile more than 2^31 bytes apart (18 GB of rows)."""
    m, n, k, ld = 1100, 16390, 1400, (1 << 24) - 16
    import _fp4x
    assert _fp4x.lib().fp4x_w8a8_form(m, n, k) == 9  # 256 rows
    xq, xs = int_codes(1, m, k)
    wq, ws = int_codes(2, n, k)
    big = torch.empty((m - 1) * ld + 1408, dtype=torch.int8, device="cuda")
    x = big.as_strided((m, k), (ld, 1))
    x.copy_(xq)
    y = F.w8a8_linear(x, xs.cuda(), padded(wq), ws.cuda())
    pick = np.r_[0:20, 240:270, 1020:1100]
    want = rounder("bf16")(o8.w8a8(xq.numpy()[pick], xs.numpy()[pick], wq.numpy(), ws.numpy()))
    same(y[torch.from_numpy(pick).cuda()], want, ld)
    del big, x


def test_linear_extreme_codes(F):
    """The longest sum of the largest products fits the int32 accumulator."""
    for m, n in ((1, 16), (20, 16), (80, 32), (256, 256)):
        k = 131071
        for a, b in ((-128, -128), (-128, 127), (127, 127)):
            x = padded(torch.full((m, k), a, dtype=torch.int8))
            w = padded(torch.full((n, k), b, dtype=torch.int8))
            one = torch.ones(m, device="cuda")
            y = F.w8a8_linear(x, one, w, torch.ones(n, device="cuda"), out_dtype=torch.float32)
            assert bool((y == float(np.float32(a * b * k))).all())
    check_linear(F, 17, 40, 512, "f32", lo=-128)


def test_linear_layouts(F):
    xq, xs = int_codes(1, 20, 200)
    wq, ws = int_codes(2, 50, 200)
    want = rounder("bf16")(o8.w8a8(xq.numpy(), xs.numpy(), wq.numpy(), ws.numpy()))
    x, w, xs, ws = xq.cuda(), wq.cuda(), xs.cuda(), ws.cuda()
    same(F.w8a8_linear(x, xs, w, ws), want, "rows off 16 bytes are copied")
    same(F.w8a8_linear(x, xs[:, None], w, ws[:, None]), want, "scales as columns")
    same(F.w8a8_linear(x.t().contiguous().t(), xs, w.t().contiguous().t(), ws), want, "column-major codes")
    big = torch.full((40, 320), 99, dtype=torch.int8, device="cuda")
    big[::2, 64:264] = x
    same(F.w8a8_linear(big[::2, 64:264], torch.stack([xs, xs], 1)[:, 0], w, ws), want, "strided rows and scales")
    bias = torch.randn(50, device="cuda").bfloat16()
    y = o8.w8a8(xq.numpy(), xs.cpu().numpy(), wq.numpy(), ws.cpu().numpy(), bias.float().cpu().numpy())
    same(F.w8a8_linear(x, xs, w, ws, bias), rounder("bf16")(y), "a bf16 bias")
    # the last row ends its storage inside a chunk of 16
    short = torch.full((16 * 19 + 9 + 16,), 7, dtype=torch.int8, device="cuda")[:16 * 19 + 9]
    s9 = short.as_strided((20, 9), (16, 1))
    y = F.w8a8_linear(s9, xs, torch.ones((5, 9), dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda"),
                      out_dtype=torch.float32)
    assert bool((y == (63 * xs)[:, None]).all())


def test_linear_bad_rows_stay_alone(F):
    """A token with NaN gives NaN in its own row and nothing else."""
    x, w = rows(1, 40, 640, "bf16"), rows(2, 100, 640, "bf16", 0.02)
    x[13, 5] = float("nan")
    x[39, 0] = float("inf")
    xq, xs = F.quantize_q8(x.cuda())
    wq, ws = F.quantize_q8(w.cuda())
    y = F.w8a8_linear(xq, xs, wq, ws).isnan()
    assert bool(y[13].all()) and bool(y[39].all()) and int(y.sum()) == 200


def test_linear_output_past_32_bits(F):
    """Output offsets past 2^31 elements."""
    m, n, k = 70000, 32768, 16
    x = torch.ones((m, k), dtype=torch.int8, device="cuda")
    w = torch.arange(n, device="cuda").remainder(100).to(torch.int8)[:, None].expand(n, k).contiguous()
    xs = torch.arange(m, device="cuda").float()
    y = F.w8a8_linear(x, xs, w, torch.ones(n, device="cuda"))
    for r in (0, 1, 65535, 65536, 69999):
        assert torch.equal(y[r], (16.0 * w[:, 0].float() * r).bfloat16()), r
    del y


def test_empty(F):
    e = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda").bfloat16()
    for fmt, ss in (("int8", (0,)), ("e4m3", (0,)), ("mx8", (0, 2))):
        q, s, h, y = F.rms_norm_q8(e, w, residual=e, fmt=fmt, normed=True)
        assert q.shape == h.shape == y.shape == (0, 64) and s.shape == ss
    q, s = F.silu_mul_q8(e)
    assert q.shape == (0, 32)
    q, s = F.quantize_q8(e)
    wq, ws = F.quantize_q8(torch.ones((5, 64), device="cuda"))
    assert F.w8a8_linear(q, s, wq, ws).shape == (0, 5)


def block(F, x, r, w, wq, ws, dq, ds):
    q, s, h = F.rms_norm_q8(x, w, residual=r)
    gu = F.w8a8_linear(q, s, wq, ws)
    return F.w8a8_linear(*F.silu_mul_q8(gu), dq, ds), h


def block_inputs(F, m, seed=0):
    x, r = rows(seed, m, 256, "bf16").cuda(), rows(seed + 1, m, 256, "bf16").cuda()
    w = torch.ones(256).bfloat16().cuda()
    return (x, r, w, *F.quantize_q8(rows(8, 2 * 160, 256, "bf16", 0.05).cuda()),
            *F.quantize_q8(rows(9, 256, 160, "bf16", 0.05).cuda()))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_graph_replays(F, m):
    a = block_inputs(F, m)
    want = [t.clone() for t in block(F, *a)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = block(F, *a)
    x0 = a[0].clone()
    for i in range(4):
        a[0].copy_(x0 if i % 2 == 0 else -x0)
        if i % 2:
            want2 = [t.clone() for t in block(F, *a)]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want2 if i % 2 else want))


def test_side_stream(F):
    a = block_inputs(F, 70)
    want = block(F, *a)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = block(F, *a)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_outputs_are_released(F):
    """Outputs are held by their callers alone, after calls that raise too."""
    import sys
    x, r = rows(1, 64, 2571, "bf16").cuda(), rows(2, 64, 2571, "bf16").cuda()
    w = torch.ones(2571).bfloat16().cuda()

    def once():
        q, s, h, y = F.rms_norm_q8(x, w, residual=r, normed=True)
        z = F.w8a8_linear(q, s, q, s)
        g = F.silu_mul_q8(x, r, "e4m3")
        for bad in (lambda: F.rms_norm_q8(x, w, residual=r, eps=-1.0), lambda: F.w8a8_linear(q, s, q, s[:1])):
            with pytest.raises(ValueError):
                bad()
        return [sys.getrefcount(t) for t in (q, s, h, y, z, *g)]
    counts = once()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(50):
        assert once() == counts
    assert max(counts) <= 4                          # the variable, the list's or tuple's entry, the argument
    assert torch.cuda.memory_allocated() == before


def test_norm_into_its_own_rows(F):
    """The next residual may be written over the residual, or over x."""
    for h in (17, 512, 2571, 9001):
        x, r, w = rows(3, 70, h, "bf16").cuda(), rows(4, 70, h, "bf16").cuda(), torch.ones(h).bfloat16().cuda()
        want = F.rms_norm_q8(x, w, residual=r)
        for over in (0, 1):
            a, b = x.clone(), r.clone()
            got = F.rms_norm_q8(a, w, residual=b, residual_out=b if over else a)
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_refusals_on_device(F):
    x = torch.ones((2, 64), device="cuda").bfloat16()
    w = torch.ones(64, device="cuda").bfloat16()
    q, s = F.quantize_q8(x)
    for call, err in (
            (lambda: F.rms_norm_q8(x, w[:63]), ValueError),
            (lambda: F.rms_norm_q8(x, w, residual=x[:1]), ValueError),
            (lambda: F.rms_norm_q8(x, w, residual=x.half()), ValueError),
            (lambda: F.rms_norm_q8(x, w.half()), ValueError),
            (lambda: F.rms_norm_q8(x, w, residual_out=x), ValueError),
            (lambda: F.rms_norm_q8(x, w, residual=x, residual_out=x[:1]), ValueError),
            (lambda: F.rms_norm_q8(x, w, eps=-1.0), ValueError),
            (lambda: F.rms_norm_q8(x, w, eps=float("nan")), ValueError),
            (lambda: F.rms_norm_q8(x, w, fmt="int4"), ValueError),
            (lambda: F.rms_norm_q8(x, w, fmt=1), ValueError),
            (lambda: F.rms_norm_q8(x, w, eps="a"), TypeError),
            (lambda: F.rms_norm_q8(x, w, w_offset=None), TypeError),
            (lambda: F.rms_norm_q8(x, w, residual=x, residual_out=x.cpu()), RuntimeError),
            (lambda: F.silu_mul_q8(x, x.cpu()), RuntimeError),
            (lambda: F.w8a8_linear(q, s, q, s, out_dtype="bf16"), TypeError),
            (lambda: F.rms_norm_q8(x.double(), w), TypeError),
            (lambda: F.rms_norm_q8(x[0], w), ValueError),
            (lambda: F.rms_norm_q8(x, w.cpu()), RuntimeError),
            (lambda: F.quantize_q8(x[:, :40].contiguous(), "mx8"), ValueError),
            (lambda: F.quantize_q8(torch.ones((1, 32769), device="cuda")), ValueError),
            (lambda: F.silu_mul_q8(x[:, :63]), ValueError),
            (lambda: F.silu_mul_q8(x, x.half()), ValueError),
            (lambda: F.silu_mul_q8(x, x[:1]), ValueError),
            (lambda: F.w8a8_linear(q.float(), s, q, s), TypeError),
            (lambda: F.w8a8_linear(q, s[:1], q, s), ValueError),
            (lambda: F.w8a8_linear(q, s, q, s.half()), ValueError),
            (lambda: F.w8a8_linear(q, s, q[:, :48], s), ValueError),
            (lambda: F.w8a8_linear(q, s, q, s, bias=s[:1]), ValueError),
            (lambda: F.w8a8_linear(q, s, q, s, out_dtype=torch.int32), TypeError),
            (lambda: F.w8a8_linear(q, s, q.cpu(), s), RuntimeError),
            (lambda: F.w8a8_linear(torch.ones((1, 131072), dtype=torch.int8, device="cuda"), s[:1],
                                   torch.ones((1, 131072), dtype=torch.int8, device="cuda"), s[:1]), ValueError)):
        with pytest.raises(err):
            call()


@pytest.mark.parametrize("tokens", [1, 37, 1024])
def test_example_block(F, tokens):
    """examples/mlp_w8a8.py against the block in fp32.  int8 codes are off by at most half a step of amax / 127: an rms of
    0.29 / 127 amax, and a row of 2560 (640) normal values has amax of about 3.6 (3.2) sigma, so each quantized operand
    adds 0.8% (0.7%) of noise: twice for the first product (inputs and weights: 1.2%), which its gate and its square
    term pass on at most doubled, and twice for the second (1.1%): 2.7%.  Rows and channels vary: 4%."""
    import importlib.util
    import os
    spec = importlib.util.spec_from_file_location(
        "mlp_w8a8", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "mlp_w8a8.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    weights, x, residual = ex.make(tokens, seed=tokens)
    y, h = ex.GatedMLP(*weights)(x, residual)
    want, h32 = ex.reference(x, residual, *weights)
    assert torch.equal(h, h32)
    assert float((y.float() - want).norm() / want.norm()) < 0.04
