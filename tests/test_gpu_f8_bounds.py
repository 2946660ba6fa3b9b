"""What the products of e4m3 codes may be off by, at the codes that make it most:
16-bit outputs are sums of the matrix cores' fp8 instruction, which cuts products
beside a larger one, and fp32 outputs of exact products (csrc/fp4x_f8.h)."""
import numpy as np
import pytest
import torch

from oracle import f8 as o
from oracle import formats as fm
from test_gpu_f8 import DT, check

pytestmark = pytest.mark.gpu

# The smallest tiles, the ring of several strips, large tiles; a K of whole blocks and one that ends inside a block.
SIZES = [(3, 48, 256), (17, 130, 384), (40, 300, 200), (260, 700, 256), (600, 1200, 300), (2100, 2304, 128)]


@pytest.fixture(scope="module")
def F(gpu):
    import fp4x_kernels
    return fp4x_kernels


def encode(v):
    q = fm.e4m3_encode(np.asarray(v, np.float32), saturate=True).astype(np.uint8)
    assert np.array_equal(fm.e4m3_decode(q), v)      # the values are ones that the format holds
    return q


def swamped(m, n, k, rng):
    """One product of 1 among eight whose others are under 2^-13 of it: all of those may be lost, all of one sign."""
    x, w = np.full((m, k), 1.875 * 2.0 ** -6), np.full((n, k), 2.0 ** -8)
    x[:, 5::8] = w[:, 5::8] = 1.0
    return x, w


def cancelling(m, n, k, rng):
    """The largest two of eight cancel: what is left may be lost whole."""
    x, w = np.full((m, k), 1.5), np.full((n, k), 2.0 ** -3)
    x[:, 2::8] = x[:, 7::8] = w[:, 2::8] = 256.0
    w[:, 7::8] = -256.0
    return x, w


def one_large_group(m, n, k, rng):
    """The largest product that there is, once in a block, far from most of the others: it cuts its own eight only."""
    x, w = rng.choice([0.5, 1.0, 1.5, -1.25], (m, k)), rng.choice([0.5, 1.0, -0.75, 1.75], (n, k))
    x[:, 19::128] = w[:, 19::128] = 448.0
    return x, w


def outlier_channels(m, n, k, rng):
    """A few channels hundreds of times larger than the rest, of either sign, as activations have them."""
    grid = fm.e4m3_decode(np.arange(256, dtype=np.uint8))
    grid = grid[np.isfinite(grid) & (np.abs(grid) < 0.5)]
    x, w = rng.choice(grid, (m, k)), rng.choice(grid, (n, k))
    at = rng.choice(k, max(1, k // 40), replace=False)
    x[:, at] = rng.choice([416.0, -384.0, 240.0], (m, len(at)))
    return x, w


PATTERNS = [swamped, cancelling, one_large_group, outlier_channels]


def operands(pattern, m, n, k):
    rng = np.random.default_rng(m + n + k)
    x, w = pattern(m, n, k, rng)
    xq, wq = encode(x), encode(w)
    kb = -(-k // 128)
    xs, ws = np.exp2(rng.integers(-2, 3, (m, kb))).astype(np.float32), np.exp2(rng.integers(-2, 3, (-(-n // 128), kb))).astype(np.float32)

    def dev(q):
        t = torch.full((q.shape[0], -(-k // 16) * 16), 0x7f, dtype=torch.uint8)
        t[:, :k] = torch.from_numpy(q)
        return t.cuda().view(torch.float8_e4m3fn)[:, :k]
    if pattern is not one_large_group:               # sums within fp16's range
        xs = xs / 64
        if pattern is cancelling or pattern is outlier_channels:
            ws = ws / 16
    else:
        xs = xs / 4096
    return (xq, xs, wq, ws), (dev(xq), torch.from_numpy(xs).t().contiguous().cuda().t(), dev(wq), torch.from_numpy(ws).cuda())


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("pattern", PATTERNS, ids=lambda p: p.__name__)
def test_products(F, pattern, m, n, k):
    """oracle.f8.linear's bounds: 7 * 2^-13 of the largest product of each eight for 16-bit outputs, fp32's roundings for fp32."""
    host, dev = operands(pattern, m, n, k)
    exact, tight = o.linear(*host)
    _, loose = o.linear(*host, cut=True)
    assert np.abs(exact).max() < 6e4                 # (fp16 holds them)
    check(F.f8_linear(*dev, out_dtype=torch.float32), exact, tight, "f32")
    for out in ("bf16", "f16"):
        check(F.f8_linear(*dev, out_dtype=DT[out]), exact, loose, out)


@pytest.mark.parametrize("pattern", PATTERNS, ids=lambda p: p.__name__)
@pytest.mark.parametrize("t,e,n,k", [(3, 40, 96, 256), (150, 5, 320, 384), (900, 3, 512, 200)])
def test_products_over_experts(F, pattern, t, e, n, k):
    host, dev = operands(pattern, t, n, k)
    xq, xs, wq, ws = dev
    ids = torch.arange(2 * t, device="cuda").view(t, 2) % e
    offsets, tokens, _ = F.expert_sort(ids, e)
    we, se = torch.stack([wq.view(torch.uint8)] * e).view(wq.dtype), torch.stack([ws] * e)
    pick = tokens.cpu().numpy()
    exact, tight = o.linear(*host)
    _, loose = o.linear(*host, cut=True)
    check(F.f8_linear_experts(xq, xs, we, se, offsets, tokens, out_dtype=torch.float32), exact[pick], tight[pick], "f32")
    for out in ("bf16", "f16"):
        check(F.f8_linear_experts(xq, xs, we, se, offsets, tokens, out_dtype=DT[out]), exact[pick], loose[pick], out)


def test_worst_of_16_bits(F):
    """The bound is no looser than what happens: where one product of eight hides the other seven, 16-bit outputs are
    short by all of them, 8.0e-4 of the sum of magnitudes and more than half a step of fp16; fp32 outputs are exact."""
    host, dev = operands(swamped, 64, 64, 256)
    exact, _ = o.linear(*host)
    assert np.array_equal(F.f8_linear(*dev, out_dtype=torch.float32).double().cpu().numpy(), exact)
    lost = exact - F.f8_linear(*dev, out_dtype=torch.float16).double().cpu().numpy()
    part = 7 * 1.875 * 2.0 ** -14 / (1 + 7 * 1.875 * 2.0 ** -14)
    assert (np.abs(lost - part * exact) <= 2.0 ** -11 * exact).all() and part > 2.0 ** -11
