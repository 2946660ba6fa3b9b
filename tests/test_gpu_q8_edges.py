"""The 8-bit activation path on the GPU, at its edges: what outputs keep alive,
rows past the grid, code rows that end their storage, and whole k-tiles in every
form of the product.  Results equal the definition bit for bit."""
import numpy as np
import pytest
import torch

from oracle import q8 as o8
from oracle.formats import e4m3_decode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F(gpu):
    import fp4x_kernels
    return fp4x_kernels


def pairs(F, fmt, m, h):
    x = torch.randn((m, h), generator=torch.Generator("cuda").manual_seed(m), device="cuda").bfloat16()
    w = torch.ones(h, device="cuda").bfloat16()
    yield lambda: F.quantize_q8(x, fmt)
    yield lambda: F.silu_mul_q8(x, x, fmt)
    yield lambda: F.rms_norm_q8(x, w, fmt=fmt)


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "mx8"])
def test_codes_and_scales_are_released_alone(F, fmt):
    """Above 1 MiB neither of them holds the other's memory; below, no more than that."""
    for m, h in ((4096, 640), (1640, 640), (1740, 608), (1030, 32768)):
        for make in pairs(F, fmt, m, h):
            q, s = make()
            per = 4 * m if fmt != "mx8" else m * h // 32
            assert q.shape == (m, h) and q.stride() == (h, 1) and s.numel() * s.element_size() == per
            torch.cuda.synchronize()
            assert q.untyped_storage().nbytes() == m * h and s.untyped_storage().nbytes() == per
            before = torch.cuda.memory_allocated()
            del q
            assert before - torch.cuda.memory_allocated() >= m * h
    for m, h in ((3, 2560), (512, 640), (1, 32)):
        for make in pairs(F, fmt, m, h):
            q, s = make()
            assert max(t.untyped_storage().nbytes() for t in (q, s)) <= 1 << 20


def test_padded_codes_of_many_rows(F):
    x = torch.randn((900, 2571), generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    q, s = F.quantize_q8(x)
    assert q.stride() == (2576, 1) and q.untyped_storage().nbytes() == 900 * 2576 and q.data_ptr() % 16 == 0
    amax = x.abs().amax(-1)
    want = amax / torch.full_like(amax, 127.0)
    assert torch.equal(s, want) and torch.equal(q, (x / want[:, None]).round().to(torch.int8))
    q1, s1 = F.quantize_q8(x[:100])                  # one allocation
    assert torch.equal(q1, q[:100]) and torch.equal(s1, s[:100])
    w = torch.randn((64, 2571), generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    qw, sw = F.quantize_q8(w)
    acc = (q.double() @ qw.double().t()).float()
    assert torch.equal(F.w8a8_linear(q, s, qw, sw, out_dtype=torch.float32), acc * s[:, None] * sw)


# silu(g) * u above -69 in steps of 2^-24: expf within an ulp (2), 1 + t (1), the rounded quotient (1) and two products (1
# each): v is within 6.  The scale adds its division: 7.  A code's quotient v / s adds both and its own division: 14.
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_silu_roundings(F, fmt, dt):
    step = 2.0 ** -24
    for m, f, spread in ((900, 1030, 2.0), (300, 4100, 8.0)):
        g = torch.Generator("cuda").manual_seed(m)
        gate, up = ((spread * torch.randn((m, f), generator=g, device="cuda")).clamp(-68, 68).to(dt) for _ in range(2))
        q, s = F.silu_mul_q8(gate, up, fmt)
        v = o8.silu_mul(gate.float().cpu().numpy(), up.float().cpu().numpy())
        s64 = np.abs(v).max(-1) / (127 if fmt == "int8" else 448)
        s = s.cpu().numpy().astype(np.float64)
        assert (np.abs(s - s64) <= 7 * step * s64).all()
        y = v / s[:, None]
        got = q.cpu().numpy().astype(np.float64) if fmt == "int8" else e4m3_decode(q.view(torch.uint8).cpu().numpy()).astype(np.float64)
        half = 0.5 if fmt == "int8" else np.maximum(np.abs(y) * 2.0 ** -4, 2.0 ** -10)
        assert (np.abs(got - y) <= half + 14 * step * np.abs(y)).all()


# every form with a K of whole k-tiles, with one and with several tiles per workgroup (tests/test_q8_routes_whole.py asserts
# that no kind is missing); full tiles and tiles that end at M or N
WHOLE = [(2, 48, 128), (1, 2560, 640), (1, 5449, 128), (3, 7000, 256), (16, 9779, 128), (9, 16384, 2560), (48, 520, 512), (5903, 2, 128),
         (34, 9820, 2688), (40, 9820, 2560), (34, 9820, 128), (8203, 35, 128), (100, 8200, 256), (18, 28777, 256), (96, 9332, 1280),
         (137, 23097, 512), (65, 35114, 640), (67, 38063, 640), (300, 5200, 1024), (35, 17360, 128), (250, 13310, 2560),
         (344, 16725, 640), (286, 20549, 640), (556, 12116, 1280), (325, 22293, 128), (194, 36551, 128), (476, 20646, 384),
         (4824, 2078, 384), (783, 12600, 640), (413, 13957, 128), (1100, 8192, 1024), (4121, 1424, 128), (652, 29929, 512),
         (2487, 6505, 640), (1100, 16384, 2560), (1536, 13312, 2560), (7510, 2118, 512), (1364, 9261, 256), (6621, 1864, 256),
         (668, 34914, 384), (3897, 6505, 384), (2048, 16384, 640), (1111, 16390, 1024), (61, 5250, 2816), (778, 334, 2688)]


# kinds with a K inside a k-tile that sizes of ragged M and N seldom take
RAGGED = [(258, 20721, 627), (340, 18892, 540), (695, 33195, 326), (1535, 17023, 295)]


@pytest.mark.parametrize("m,n,k", WHOLE + RAGGED)
def test_products_of_every_kind(F, m, n, k):
    g = torch.Generator("cuda").manual_seed(m + n + k)
    xq, wq = (torch.randint(-128, 128, (r, k + 15 & -16), generator=g, device="cuda", dtype=torch.int8)[:, :k] for r in (m, n))
    xs, ws, b = (0.5 + torch.rand(r, generator=g, device="cuda") for r in (m, n, n))
    acc = (xq.double() @ wq.double().t()).float()    # the exact sum, rounded once
    y = (acc * xs[:, None]) * ws
    for _ in range(3):
        assert torch.equal(F.w8a8_linear(xq, xs, wq, ws, b, torch.float32), y + b)
    assert torch.equal(F.w8a8_linear(xq, xs, wq, ws), y.bfloat16())
    assert torch.equal(F.w8a8_linear(xq, xs, wq, ws, out_dtype=torch.float16).view(torch.int16), y.half().view(torch.int16))


# more rows than a grid of 2^20 workgroups takes at once: rows of a wave's part, of a wave and of several waves (2, 3 and 4
# chunks per lane), each a window of one vector, eight values on from the row before
CAP = 1 << 20
PAST = [(64 * CAP + 5, 16), (4 * CAP + 5, 264), (CAP + 3, 1032), (CAP + 1031, 1056), (CAP + 3, 4104), (CAP + 3, 24584)]


@pytest.mark.parametrize("m,h", PAST)
def test_rows_past_the_grid(F, m, h):
    g = torch.Generator("cuda").manual_seed(h)

    def windows():
        v = torch.randn(8 * m + h, generator=g, device="cuda").bfloat16()
        return v.as_strided((m, h), (8, 1))
    x, r = windows(), windows()
    w = (1 + 0.2 * torch.randn(h, generator=g, device="cuda")).bfloat16()
    at = torch.cat([torch.arange(40), torch.arange(m - 40, m), torch.linspace(0, m - 1, 40).long()]).cuda()
    cut = m // 2                                     # a call of half as many rows takes one pass

    def both(call, oracle):
        whole = call(slice(None))
        for part in (slice(0, cut), slice(cut, None)):
            for a, b in zip(whole, call(part)):
                assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8))
                           for p, q in zip(a[part].split(1 << 20), b.split(1 << 20)))
        for a, b in zip(whole, oracle):
            a = a[at].cpu()
            a = a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a.float() if a.dtype == torch.bfloat16 else a
            assert np.array_equal(a.numpy(), b)
    xs, rs = x[at].float().cpu().numpy(), r[at].float().cpu().numpy()
    fmt = "mx8" if h % 32 == 0 else "int8"
    both(lambda p: F.quantize_q8(x[p], fmt), o8.quantize(xs, fmt))
    if h > 8192:                                     # (26 GB of codes are enough)
        return
    v, n = o8.rms_norm(xs, w.float().cpu().numpy(), 1e-6, rs, lambda a: torch.from_numpy(a).bfloat16().float().numpy())
    both(lambda p: F.rms_norm_q8(x[p], w, residual=r[p], fmt=fmt), (*o8.quantize(v, fmt), n))


def copies(call):
    """A call's result and how many allocations it makes."""
    call()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    y = call()
    return y, torch.cuda.memory_stats()["allocation.all.allocated"] - before


def test_code_rows_that_end_their_storage(F):
    """The last row may end inside a chunk of 16 bytes only where the storage goes on to its end; otherwise it is copied."""
    k = 9
    w, one = torch.ones((5, k), dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda")
    wq = torch.zeros((5, 16), dtype=torch.int8, device="cuda")[:, :k]
    wq.copy_(w)
    xs = 1 + torch.arange(20, device="cuda").float()
    for end, allocations in ((16 * 19 + k, 2), (16 * 19 + 15, 2), (16 * 20, 1)):   # the output, and a copy
        flat = torch.full((end,), 7, dtype=torch.int8, device="cuda")
        assert flat.untyped_storage().nbytes() == end and flat.data_ptr() % 16 == 0
        x = flat.as_strided((20, k), (16, 1))
        y, n = copies(lambda: F.w8a8_linear(x, xs, wq, one, out_dtype=torch.float32))
        assert n == allocations and bool((y == (7 * k * xs)[:, None]).all())
        y, n = copies(lambda: F.w8a8_linear(wq, one, x, xs, out_dtype=torch.float32))   # as weights
        assert n == allocations and bool((y == (7 * k * xs)[None]).all())
    flat = torch.full((16 * 19 + k + 32,), 7, dtype=torch.int8, device="cuda")
    x = flat[32:].as_strided((20, k), (16, 1), 32)   # the same rows further on
    assert copies(lambda: F.w8a8_linear(x, xs, wq, one))[1] == 2
