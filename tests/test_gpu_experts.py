"""Experts on the GPU (csrc/fp4x_experts.hip, csrc/fp4x_f8.h): the sort equals the
oracle, rows are copied as they are, sums and gradients are within the bound of
their fp32 evaluation, and the experts' products equal the plain product of each
expert's rows."""
import numpy as np
import pytest
import torch

from oracle import f8 as o
from test_gpu_f8 import exact_operands, exact_product

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def F(gpu):
    import fp4x_kernels
    return fp4x_kernels


def route(t, k, experts, seed, drop=0.0):
    """Ids without repeats in a token where there are enough experts, some of them -1 or another rank's."""
    g = torch.Generator().manual_seed(seed)
    if k <= experts:
        ids = (torch.rand((t, experts), generator=g) + 0.3 * torch.rand(experts, generator=g)).topk(k, -1)[1]
    else:
        ids = torch.randint(0, experts, (t, k), generator=g)
    lost = torch.rand((t, k), generator=g) < drop
    return torch.where(lost, torch.where(torch.rand((t, k), generator=g) < 0.5, -1, experts + 3), ids)


SORTS = [(0, 8, 16), (1, 1, 1), (1, 8, 512), (3, 8, 512), (5, 3, 7), (64, 1, 2), (100, 6, 60), (511, 8, 128), (512, 8, 64),
         (513, 8, 512), (700, 10, 513), (4001, 8, 256), (3000, 2, 4096), (2, 300, 40), (20000, 8, 512), (33000, 4, 3000)]


@pytest.mark.parametrize("t,k,experts", SORTS)
@pytest.mark.parametrize("drop", [0.0, 0.4, 1.0])
def test_sort(F, t, k, experts, drop):
    ids = route(t, k, experts, t + k, drop)
    want = o.sort(ids.numpy(), experts)
    for v in (ids.cuda(), ids.int().cuda(), torch.nn.functional.pad(ids, (2, 1), value=0).cuda()[:, 2:2 + k], ids.t().contiguous().cuda().t()):
        for got, w in zip(F.expert_sort(v, experts), want):
            assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), w)


def test_sort_one_expert_takes_all(F):
    for t in (700, 9000):
        ids = torch.full((t, 2), 5)
        ids[::3, 1] = 1 << 40
        want = o.sort(ids.numpy(), 9)
        for got, w in zip(F.expert_sort(ids.cuda(), 9), want):
            assert np.array_equal(got.cpu().numpy(), w)


def sorted_rows(F, t, k, experts, seed, drop=0.2):
    return F.expert_sort(route(t, k, experts, seed, drop).cuda(), experts)


ROWS = [(1, 1, 4, 1), (3, 8, 512, 2560), (20, 3, 7, 5), (20, 3, 7, 8), (50, 4, 16, 2571), (333, 6, 60, 130), (64, 2, 8, 4097), (10, 2, 8, 9000), (1500, 8, 64, 640)]


@pytest.mark.parametrize("t,k,experts,h", ROWS)
def test_rows(F, t, k, experts, h):
    _, tokens, _ = sorted_rows(F, t, k, experts, h)
    at = tokens.long().cpu()
    for dt in (torch.bfloat16, torch.float32, torch.uint8, torch.float8_e4m3fn):
        x = (100 * torch.randn((t, h + 3), generator=torch.Generator().manual_seed(1))).to(dt)
        bits = x.view(torch.uint8).view(t, h + 3, x.element_size())
        for v, b in ((x[:, :h], bits[:, :h]), (x[:, 3:], bits[:, 3:])):
            got = F.expert_rows(v.cuda(), tokens)
            want = torch.where((at < 0)[:, None, None], 0, b[at.clamp_min(0)])
            assert got.dtype == dt and torch.equal(got.cpu().view(torch.uint8).view(len(at), h, -1), want)


def close(got, want, bound):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half
    d = np.abs(got.double().cpu().numpy() - want)
    bad = d > bound + half * (np.abs(want) + bound) + tiny
    assert not bad.any(), (int(bad.sum()), bad.size, float((d - half * np.abs(want)).max()))


@pytest.mark.parametrize("t,k,experts,h", ROWS)
@pytest.mark.parametrize("dt", list(DT))
def test_combine_and_gradient(F, t, k, experts, h, dt):
    g = torch.Generator().manual_seed(h)
    _, tokens, slots = sorted_rows(F, t, k, experts, h)
    n = int((tokens >= 0).sum())
    y = torch.randn((t * k, h + 5), generator=g).to(DT[dt])
    y[n:] = float("nan")                             # what no pair has is not read
    y = y.cuda()[:, 2:h + 2]
    dout = torch.randn((t, h), generator=g).to(DT[dt]).cuda()
    s = slots.cpu().numpy()
    yn, dn = y.float().cpu().numpy(), dout.float().cpu().numpy()
    yn[n:] = 0
    close(F.expert_combine(y, slots), *o.combine(yn, s))
    for wdt in {torch.float32, DT[dt]}:
        w = torch.rand((t, k), generator=g).to(wdt).cuda()
        wn = w.float().cpu().numpy()
        close(F.expert_combine(y, slots, w), *o.combine(yn, s, wn))
        dy, dw = F.expert_combine_grad(dout, y, slots, w, tokens)
        assert dy.dtype == y.dtype and dw.dtype == wdt and dw.shape == w.shape
        want_dy, want_dw, bound = o.combine_grad(dn, yn, s, wn)
        close(dy, want_dy, np.abs(want_dy) * 2.0 ** -24)
        close(dw, want_dw, bound)
        assert torch.equal(dy[n:], torch.zeros_like(dy[n:])) and torch.equal(dw[slots < 0], torch.zeros_like(dw[slots < 0]))


def test_gradients_against_differences(F):
    """In fp32: the sum is linear in the rows and in the weights, so a difference over any step is the gradient."""
    t, k, h = 20, 3, 130
    g = torch.Generator().manual_seed(0)
    _, tokens, slots = sorted_rows(F, t, k, 7, 3)
    y, w, dout = torch.randn((t * k, h), generator=g).cuda(), torch.rand((t, k), generator=g).cuda(), torch.randn((t, h), generator=g).cuda()
    dy, dw = F.expert_combine_grad(dout, y, slots, w, tokens)
    x = torch.randn((t, h), generator=g).cuda()
    dx = F.expert_combine(dy, slots)                 # of the rows
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        vy, vw, vx = torch.randn(y.shape, generator=g).cuda(), torch.randn(w.shape, generator=g).cuda(), torch.randn(x.shape, generator=g).cuda()

        def along(f, at, v, grad):
            up, down = (float((f(at + e * v).double() * dout.double()).sum()) for e in (0.5, -0.5))
            want = float((grad.double() * v.double()).sum())
            scale = float((grad.double() * v.double()).abs().sum())
            assert abs(up - down - want) <= 2.0 ** -18 * scale, (up - down, want)
        along(lambda v: F.expert_combine(v, slots, w), y, vy, dy)
        along(lambda v: F.expert_combine(y, slots, v), w, vw, dw)
        # rows and sum together: out = combine(rows(x)) has the gradient dx for y = rows(x)
        along(lambda v: F.expert_combine(F.expert_rows(v, tokens), slots, w), x, vx, dx)


def test_combine_more_pairs_than_experts_rows(F):
    """The same slot twice, slots past the rows, no rows at all."""
    y = torch.randn((10, 40), generator=torch.Generator().manual_seed(1)).cuda()
    slots = torch.tensor([[0, 0, 9], [10, 1 << 30, -7], [3, -1, 3]], dtype=torch.int32).cuda()
    close(F.expert_combine(y, slots), *o.combine(y.cpu().numpy(), slots.cpu().numpy()))
    assert torch.equal(F.expert_combine(y[:0], slots), torch.zeros((3, 40), device="cuda"))
    assert F.expert_combine(y, slots[:0]).shape == (0, 40)
    many = torch.arange(10, dtype=torch.int32).repeat(13).view(1, 130).cuda()
    close(F.expert_combine(y, many), *o.combine(y.cpu().numpy(), many.cpu().numpy()))


# ------------------------------------------------------------------ products
def expert_operands(rows, experts, n, k, seed):
    xq, xs, wq, ws = exact_operands(rows, experts * n, k, seed)
    nb = -(-n // 128)
    g = torch.Generator(device="cuda").manual_seed(seed)
    ws = torch.exp2(torch.randint(-2, 3, (experts, nb, ws.shape[1]), generator=g, device="cuda").float())
    whole = wq.untyped_storage()
    ld = wq.stride(0)
    w3 = torch.tensor([], dtype=torch.float8_e4m3fn, device="cuda").set_(whole, 0, (experts, n, k), (n * ld, ld, 1))
    return xq, xs, w3, ws


def plain_experts(xq, xs, wq, ws, offsets, tokens):
    out = []
    off = offsets.tolist()
    for e in range(wq.shape[0]):
        at = torch.arange(off[e], off[e + 1], device="cuda")
        if tokens is not None:
            at = tokens[at].long()
        out.append(exact_product(xq.view(torch.uint8)[at].view(torch.float8_e4m3fn), xs[at], wq[e], ws[e]))
    return torch.cat(out)


EXPERTS = [(1, 1, 1, 16, 16), (3, 8, 512, 128, 256), (3, 8, 16, 1280, 2560), (20, 4, 9, 100, 130), (50, 2, 4, 257, 300), (100, 8, 64, 300, 128),
           (200, 8, 40, 640, 500), (400, 6, 6, 256, 640), (600, 8, 128, 200, 257), (1000, 4, 3, 700, 384), (2000, 2, 5, 1280, 640), (333, 1, 300, 130, 1000),
           (64, 2, 1000, 48, 64)]


@pytest.mark.parametrize("t,k,experts,n,kk", EXPERTS)
def test_products(F, t, k, experts, n, kk):
    for drop in (0.0, 0.3):
        offsets, tokens, _ = sorted_rows(F, t, k, experts, n, drop)
        total = int(offsets[-1])
        xq, xs, wq, ws = expert_operands(t, experts, n, kk, t)
        want = plain_experts(xq, xs, wq, ws, offsets, tokens)
        for out in (torch.float32, torch.bfloat16):
            got = F.f8_linear_experts(xq, xs, wq, ws, offsets, tokens, out_dtype=out)
            assert got.shape == (t * k, n) and torch.equal(got[:total], want.float().to(out))
        xq, xs, _, _ = exact_operands(t * k, 1, kk, t + 1)
        got = F.f8_linear_experts(xq, xs, wq, ws, offsets, out_dtype=torch.float32)
        assert torch.equal(got[:total], plain_experts(xq, xs, wq, ws, offsets, None).float())


def test_rows_behind_the_last_are_left(F):
    """Through the C entry, whose output is the caller's: rows that no expert has keep what they held."""
    import _fp4x as B
    xq, xs, wq, ws = expert_operands(300, 3, 200, 256, 1)
    for off in ((0, 0, 150, 200), (7, 90, 90, 260), (0, 300, 300, 300), (5, 5, 5, 5)):
        offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
        out = torch.full((300, 200), 7.0, device="cuda")
        B.check(B.lib().fp4x_f8_linear_experts(xq.data_ptr(), xq.stride(0), xs.data_ptr(), xs.stride(0), xs.stride(1), 300, None, offsets.data_ptr(), 3,
                                               wq.data_ptr(), wq.stride(1), wq.stride(0), ws.data_ptr(), out.data_ptr(), 200, B.DT_F32, 300, 200, 256,
                                               B.stream_of(out)), "f8_linear_experts")
        want = torch.full((300, 200), 7.0, device="cuda")
        want[off[0]:off[3]] = plain_experts(xq, xs, wq, ws, offsets, None).float()
        assert torch.equal(out, want)


def test_offsets_and_tokens_are_cut(F):
    """Offsets that fall or leave the rows, tokens that are none: no other memory is touched, ordinary experts are right."""
    xq, xs, wq, ws = expert_operands(100, 4, 130, 128, 2)
    offsets = torch.tensor([0, 60, 50, 90, 1 << 30], dtype=torch.int32, device="cuda")
    got = F.f8_linear_experts(xq, xs, wq, ws, offsets, out_dtype=torch.float32)
    want = exact_product(xq, xs, wq[0], ws[0]).float()
    assert torch.equal(got[:50], want[:50])
    last = exact_product(xq, xs, wq[3], ws[3]).float()
    assert torch.equal(got[90:], last[90:])
    offsets = torch.tensor([0, 3, 3, 3, 5], dtype=torch.int32, device="cuda")
    tokens = torch.tensor([99, 1 << 30, 2, -5, 4], dtype=torch.int32, device="cuda")
    got = F.f8_linear_experts(xq, xs, wq, ws, offsets, tokens, out_dtype=torch.float32)
    assert torch.equal(got[:3], want[[99, 99, 2]]) and torch.equal(got[3:], last[[0, 4]])


def test_block(F):
    """A block of experts as a server runs it, against fp64 of the same codes at each stage."""
    t, k, experts, hidden, inner = 70, 4, 12, 640, 384
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn((t, hidden), generator=g, device="cuda").bfloat16()
    res = torch.randn((t, hidden), generator=g, device="cuda").bfloat16()
    gate_up = F.quantize_f8(0.05 * torch.randn((experts, 2 * inner, hidden), generator=g, device="cuda"))
    down = F.quantize_f8(0.05 * torch.randn((experts, hidden, inner), generator=g, device="cuda"))
    norm = torch.ones(hidden, device="cuda").bfloat16()
    router = torch.randn((experts, hidden), generator=g, device="cuda") / hidden ** 0.5

    def block():
        q, s, h, v = F.rms_norm_q8(x, norm, residual=res, fmt="e4m3_g128", normed=True)
        w, ids = torch.softmax(v.float() @ router.t(), -1).topk(k, -1)
        offsets, tokens, slots = F.expert_sort(ids, experts)
        a = F.f8_linear_experts(q, s, *gate_up, offsets, tokens, out_dtype=torch.bfloat16)
        aq, as_ = F.silu_mul_q8(a, fmt="e4m3_g128")
        y = F.f8_linear_experts(aq, as_, *down, offsets, out_dtype=torch.bfloat16)
        return F.expert_combine(y, slots, w), h, (q, s, offsets, tokens, slots, a, aq, as_, y, w)
    out, h, (q, s, offsets, tokens, slots, a, aq, as_, y, w) = block()
    assert torch.equal(h, (x.float() + res.float()).bfloat16())
    off, tok = offsets.tolist(), tokens.cpu().numpy()

    def stage(got, cq, cs, weight, pick):
        for e in range(experts):
            at = slice(off[e], off[e + 1])
            rows = tok[at] if pick else np.arange(off[e], off[e + 1])
            want, bound = o.linear(cq.view(torch.uint8).cpu().numpy()[rows], cs.cpu().numpy()[rows], weight[0][e].view(torch.uint8).cpu().numpy(),
                                   weight[1][e].cpu().numpy(), cut=True)
            close(got[at], want, bound)
    stage(a, q, s, gate_up, True)
    stage(y, aq, as_, down, False)
    close(out, *o.combine(y.float().cpu().numpy(), slots.cpu().numpy(), w.cpu().numpy()))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, _, _ = block()
    for seed in range(3):
        x.copy_(torch.randn((t, hidden), generator=g, device="cuda").bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        eager, _, _ = block()
        assert torch.equal(captured, eager)
