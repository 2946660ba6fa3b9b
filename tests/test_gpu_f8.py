"""e4m3 with a scale per block of 128 on the GPU (csrc/fp4x_rowq.hip,
csrc/fp4x_f8.h): rows and weights equal the oracle bit for bit; products are
within the bound of their fp32 evaluation."""
import numpy as np
import pytest
import torch

from oracle import f8 as o
from oracle import formats as fm
from oracle import q8 as o8

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FMT = "e4m3_g128"


@pytest.fixture(scope="module")
def F(gpu):
    import fp4x_kernels
    return fp4x_kernels


def u8(t):
    return t.view(torch.uint8).cpu().numpy()


def rows(m, h, dt, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((m, h), generator=g) * torch.exp(spread * torch.randn((m, 1), generator=g))).to(DT[dt])


def same_rows(q, s, v):
    want_q, want_s = o.quantize_rows(v)
    assert q.dtype == torch.float8_e4m3fn and q.shape == v.shape and s.shape == want_s.shape
    assert np.array_equal(s.cpu().numpy().view(np.uint32) & 0x7fffffff, want_s.view(np.uint32) & 0x7fffffff)
    assert np.array_equal(u8(q), want_q)


SIZES = [(1, 1), (3, 5), (2, 8), (5, 31), (4, 64), (3, 100), (7, 127), (2, 128), (3, 129), (9, 250), (2, 256), (3, 257),
         (1, 640), (300, 640), (5, 1000), (3, 2560), (777, 2571), (6, 6145), (5000, 130), (2, 8199), (4, 16385), (2, 32768)]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,h", SIZES)
def test_rows(F, m, h, dt):
    x = rows(m, h, dt, m + h)
    q, s = F.quantize_q8(x.cuda(), FMT)
    line = -(-h // 128) * 128                        # rows start on a line where that adds a sixteenth at most
    assert q.stride(0) == (line if (line - h) * 16 <= h else -(-h // 16) * 16) or m == 1
    same_rows(q, s, x.float().numpy())


@pytest.mark.parametrize("m,h", [(1, 7), (3, 130), (3, 2560), (333, 2571), (2100, 640), (3, 12000)])
@pytest.mark.parametrize("rdt", [None, "bf16", "f32"])
def test_norm(F, m, h, rdt):
    x, r = rows(m, h, "bf16", h), None if rdt is None else rows(m, h, rdt, h + 1)
    w = (1 + 0.2 * torch.randn(h, generator=torch.Generator().manual_seed(2))).bfloat16()
    got = F.rms_norm_q8(x.cuda(), w.cuda(), residual=None if r is None else r.cuda(), fmt=FMT, normed=True)
    back = (lambda a: torch.from_numpy(a).to(r.dtype).float().numpy()) if r is not None else None
    v, hr = o8.rms_norm(x.float().numpy(), w.float().numpy(), 1e-6, None if r is None else r.float().numpy(), back)
    same_rows(got[0], got[1], v)
    if r is not None:
        assert np.array_equal(got[2].float().cpu().numpy(), hr)
    assert torch.equal(got[-1].cpu(), torch.from_numpy(v).bfloat16())


# silu(g) * u: within 6 steps of 2^-24 above -69 (expf 2, 1 + t 1, the quotient 1, two products), the scale 7, a code's
# quotient 14, as for the formats with one scale per row.
@pytest.mark.parametrize("m,f", [(3, 640), (900, 1030), (2, 100), (300, 4100)])
def test_silu(F, m, f):
    step = 2.0 ** -24
    g = torch.Generator().manual_seed(f)
    gu = (2 * torch.randn((m, 2 * f), generator=g)).clamp(-68, 68).bfloat16()
    q, s = F.silu_mul_q8(gu.cuda(), fmt=FMT)
    v = o8.silu_mul(gu[:, :f].float().numpy(), gu[:, f:].float().numpy())
    codes, s = fm.e4m3_decode(u8(q)).astype(np.float64), s.cpu().numpy().astype(np.float64)
    for b in range(s.shape[1]):
        at = slice(128 * b, 128 * b + 128)
        s64 = np.abs(v[:, at]).max(-1) / 448
        assert (np.abs(s[:, b] - s64) <= 7 * step * s64).all()
        y = v[:, at] / s[:, b:b + 1]
        assert (np.abs(codes[:, at] - y) <= np.maximum(np.abs(y) * 2.0 ** -4, 2.0 ** -10) + 14 * step * np.abs(y)).all()


def test_rows_strides_and_bad_values(F):
    x = rows(40, 700, "f32", 5)
    x[3, 130] = float("inf")
    x[4, 699] = float("nan")
    x[5, :128] = 0
    x[6, 128:256] = 1e-30
    x[7, 0:128] = 3e38
    want = x.clone()
    same_rows(*F.quantize_q8(x.cuda(), FMT), want.numpy())
    big = torch.zeros((40, 903))
    big[:, 101:801] = x
    same_rows(*F.quantize_q8(big.cuda()[:, 101:801], FMT), want.numpy())
    same_rows(*F.quantize_q8(x.t().contiguous().cuda().t(), FMT), want.numpy())
    q, s = F.quantize_q8(x.cuda()[:0], FMT)
    assert q.shape == (0, 700) and s.shape == (0, 6)


def test_scales_lie_by_block(F):
    for m, h in ((5, 700), (3000, 2560)):            # one allocation, and one each
        q, s = F.quantize_q8(rows(m, h, "bf16", 1).cuda(), FMT)
        assert s.shape == (m, -(-h // 128)) and s.stride() == (1, m) and s.dtype == torch.float32


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (128, 128), (130, 257), (300, 1000), (640, 2560), (3, 40, 200), (2, 257, 129)])
def test_weight(F, shape, dt):
    w = (0.02 * torch.randn(shape, generator=torch.Generator().manual_seed(shape[-1]))).to(DT[dt])
    q, s = F.quantize_f8(w.cuda())
    assert q.shape == w.shape and q.dtype == torch.float8_e4m3fn and q.stride(-2) % 16 == 0
    w2, q2, s2 = (t if t.dim() == 3 else t[None] for t in (w, q, s))
    for e in range(len(w2)):
        want_q, want_s = o.quantize_weight(w2[e].float().numpy())
        assert np.array_equal(s2[e].cpu().numpy(), want_s) and np.array_equal(u8(q2[e]), want_q)


def test_weight_strides_and_bad_values(F):
    w = 0.02 * torch.randn((200, 300), generator=torch.Generator().manual_seed(1))
    w[130, 5] = float("nan")
    w[0, 299] = -float("inf")
    want_q, want_s = o.quantize_weight(w.numpy())
    for v in (w.cuda(), w.t().contiguous().cuda().t(), torch.nn.functional.pad(w, (1, 6)).cuda()[:, 1:301]):
        q, s = F.quantize_f8(v)
        assert np.array_equal(u8(q), want_q)
        got = s.cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want_s)) and np.array_equal(got[~np.isnan(got)], want_s[~np.isnan(want_s)])


# ------------------------------------------------------------------ the product
def operands(m, n, k, seed, device="cuda"):
    """Codes and scales with bytes behind each row's end that are NaN codes, and the same in numpy."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)))).astype(np.float32)
    w = (0.02 * rng.standard_normal((n, k))).astype(np.float32)
    (xq, xs), (wq, ws) = o.quantize_rows(x), o.quantize_weight(w)

    def dev(q):
        t = torch.full((q.shape[0], -(-k // 16) * 16), 0x7f, dtype=torch.uint8)
        t[:, :k] = torch.from_numpy(q)
        return t.to(device).view(torch.float8_e4m3fn)[:, :k]
    return (xq, xs, wq, ws), (dev(xq), torch.from_numpy(xs).t().contiguous().to(device).t(), dev(wq), torch.from_numpy(ws).to(device))


def check(got, want, bound, out):
    got = got.double().cpu().numpy()
    half = torch.finfo(DT[out]).eps / 2
    tiny = torch.finfo(DT[out]).smallest_normal * half
    d = np.abs(got - want)
    bad = d > bound + half * (np.abs(want) + bound) + tiny
    assert not bad.any(), (int(bad.sum()), bad.size, float((d / (bound + half * np.abs(want) + tiny)).max()))


LINEAR = [(1, 1, 1), (1, 16, 16), (3, 100, 128), (2, 130, 129), (3, 2560, 640), (16, 1280, 2560), (17, 300, 250), (33, 129, 384),
          (64, 640, 1000), (65, 1000, 513), (128, 256, 256), (200, 384, 300), (250, 1331, 2500), (300, 2560, 640),
          (513, 700, 120), (1000, 1300, 257), (2, 16400, 2560), (100, 2560, 6144), (1, 640, 20000)]


@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear(F, m, n, k):
    host, dev = operands(m, n, k, m + n + k)
    for out in DT:
        want, bound = o.linear(*host, cut=out != "f32")
        check(F.f8_linear(*dev, out_dtype=DT[out]), want, bound, out)
    bias = np.random.default_rng(1).standard_normal(n).astype(np.float32)
    want, bound = o.linear(*host, bias)
    check(F.f8_linear(*dev, bias=torch.from_numpy(bias).cuda(), out_dtype=torch.float32), want, bound, "f32")


def exact_operands(m, n, k, seed):
    """Codes of small whole numbers and scales of powers of two: every sum is exact in fp32, in any order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kb = -(-k // 128)

    def codes(r):
        t = torch.full((r, -(-k // 16) * 16), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :k]
        t.copy_(torch.randint(-4, 5, (r, k), generator=g, device="cuda").float())
        return t

    def powers(*shape):
        return torch.exp2(torch.randint(-2, 3, shape, generator=g, device="cuda").float())
    return codes(m), powers(kb, m).t(), codes(n), powers(-(-n // 128), kb)


def exact_product(xq, xs, wq, ws):
    """In fp64 on the GPU, exact for exact_operands."""
    k, n = xq.shape[1], wq.shape[0]
    x = xq.double() * xs.double().repeat_interleave(128, 1)[:, :k]
    w = wq.double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return x @ w.t()


# sums stay below 16 x 16 x 10240 x 2^4 / 2^-4 units: 2^23.4 at the most, and these are far from the most
@pytest.mark.parametrize("m,n,k", [(1, 2560, 640), (16, 16384, 2560), (64, 2560, 6144), (250, 13310, 2500), (512, 2560, 640),
                                   (1024, 4096, 1024), (2048, 16384, 384), (4096, 16384, 2560), (4000, 9999, 1111), (70000, 130, 257),
                                   (700, 18000, 130), (3000, 3000, 129)])
def test_linear_exact(F, m, n, k):
    ops = exact_operands(m, n, k, m + k)
    bias = torch.randint(-100, 101, (n,), device="cuda").float()
    want = exact_product(*ops)
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(F.f8_linear(*ops, out_dtype=out), want.float().to(out))
    assert torch.equal(F.f8_linear(*ops, bias=bias, out_dtype=torch.float32), (want + bias.double()).float())


def test_linear_strides_and_layouts(F):
    ops = exact_operands(70, 200, 300, 3)
    want = exact_product(*ops).float()
    xq, xs, wq, ws = ops
    alike = [(xq, xs.contiguous(), wq, ws),
             (xq.contiguous(), xs, wq.contiguous(), ws),                   # 300 bytes a row: copied
             (xq, xs, wq, ws.t().contiguous().t()),
             (xq, torch.nn.functional.pad(xs, (1, 2))[:, 1:4], wq, ws),
             (xq.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn), xs, wq, ws)]
    for a in alike:
        assert torch.equal(F.f8_linear(*a, out_dtype=torch.float32), want)
    one = F.f8_linear(xq, xs[:, :1].expand(-1, 3), wq, ws, out_dtype=torch.float32)   # a stride of 0
    assert torch.equal(one, exact_product(xq, xs[:, :1].expand(-1, 3), wq, ws).float())
    assert F.f8_linear(xq[:0], xs[:0], wq, ws).shape == (0, 200)


def test_bad_rows_stay_alone(F):
    xq, xs, wq, ws = exact_operands(200, 300, 400, 7)
    want = exact_product(xq, xs, wq, ws).float()
    xs = xs.clone()
    xs[3, 1] = float("nan")
    xs[150, 3] = float("inf")
    got = F.f8_linear(xq, xs, wq, ws, out_dtype=torch.float32)
    good = [m for m in range(200) if m not in (3, 150)]
    assert torch.equal(got[good], want[good]) and got[3].isnan().all() and not got[150].isfinite().any()
    ws = ws.clone()
    ws[2, 0] = float("nan")                          # columns 256 to 299
    got = F.f8_linear(xq[good], xs[good], wq, ws, out_dtype=torch.float32)
    assert torch.equal(got[:, :256], want[good][:, :256]) and got[:, 256:].isnan().all()


def test_end_to_end_error(F):
    """Rows and weights quantized, multiplied: 2^-4 relative a value on each side, averaged over 2560 products."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x, w = torch.randn((300, 2560), generator=g, device="cuda").bfloat16(), (0.02 * torch.randn((640, 2560), generator=g, device="cuda")).bfloat16()
    y = F.f8_linear(*F.quantize_q8(x, FMT), *F.quantize_f8(w), out_dtype=torch.float32)
    want = x.double() @ w.double().t()
    assert float((y.double() - want).norm() / want.norm()) < 2 * 2.0 ** -4


def test_graph_and_stream(F):
    ops = exact_operands(100, 640, 1000, 1)
    x = torch.randn((100, 1000), device="cuda")
    xq, xs = F.quantize_q8(x, FMT)
    F.f8_linear(xq, xs, *ops[2:])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gq, gs = F.quantize_q8(x, FMT)
        gy = F.f8_linear(gq, gs, *ops[2:])
    side = torch.cuda.Stream()
    for i in range(3):
        x.copy_(torch.randn((100, 1000), generator=torch.Generator("cuda").manual_seed(i), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            q, s = F.quantize_q8(x, FMT)
            y = F.f8_linear(q, s, *ops[2:])
        side.synchronize()
        assert torch.equal(gq.view(torch.uint8), q.view(torch.uint8)) and torch.equal(gs, s) and torch.equal(gy, y)
