"""Calls of the operators on e4m3 blocks and experts as a program makes them:
what is refused, captured calls replayed with eager work between, streams at
once, rows past 2^31 elements, and the example's gradients."""
import importlib.util
import os

import pytest
import torch

from oracle import f8 as o
from test_gpu_experts import expert_operands, plain_experts
from test_gpu_experts import route as host_route
from test_gpu_f8 import FMT, exact_operands, exact_product

pytestmark = pytest.mark.gpu


def route(*a, **kw):
    return host_route(*a, **kw).cuda()


@pytest.fixture(scope="module")
def F(gpu):
    import fp4x_kernels
    return fp4x_kernels


def test_refusals(F):
    xq, xs, wq, ws = exact_operands(6, 300, 400, 0)
    eq, es = wq[None].expand(2, -1, -1), ws[None].expand(2, -1, -1).contiguous()
    off = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    tok = torch.zeros(6, dtype=torch.int32, device="cuda")
    f8 = torch.float8_e4m3fn
    long = torch.zeros((2, 131072), device="cuda").to(f8)
    wide = torch.zeros((2, 1024), device="cuda")
    x = torch.ones((6, 64), device="cuda")
    ids = torch.zeros((3, 2), dtype=torch.int64, device="cuda")
    slots = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    w = torch.ones((3, 2), device="cuda")
    lin, ex, srt, rws, cmb, grd = F.f8_linear, F.f8_linear_experts, F.expert_sort, F.expert_rows, F.expert_combine, F.expert_combine_grad
    bad = [
        (lin, xq.cpu(), xs, wq, ws), (lin, xq, xs.cpu(), wq, ws), (lin, xq, xs, wq.cpu(), ws), (lin, xq, xs, wq, ws.cpu()),
        (lin, xq.view(torch.uint8), xs, wq, ws), (lin, xq, xs.half(), wq, ws), (lin, xq, xs, wq.view(torch.int8), ws), (lin, xq, xs, wq, ws.double()),
        (lin, xq[0], xs, wq, ws), (lin, xq, xs[:5], wq, ws), (lin, xq, xs[:, :3], wq, ws), (lin, xq, xs, wq, ws[:2]), (lin, xq, xs, wq, ws[:, :1]),
        (lin, xq[:, :384], xs[:, :3], wq, ws), (lin, xq, xs, eq, es), (lin, xq, xs, wq, ws, torch.ones(299, device="cuda")),
        (lin, xq, xs, wq, ws, torch.ones(300)), (lin, long, wide, long, wide[:1]), (lin, xq[:, :0], xs[:, :0], wq[:, :0], ws[:, :0]),
        (ex, xq, xs, wq, ws, off), (ex, xq, xs, eq, es, off[:2]), (ex, xq, xs, eq, es, off.long()), (ex, xq, xs, eq, es, off.cpu()),
        (ex, xq, xs, eq, es, off, tok.long()), (ex, xq, xs, eq, es, off, tok.cpu()), (ex, xq, xs, eq, es, off, tok[:, None]),
        (ex, xq[:0], xs[:0], eq, es, off, tok), (ex, xq, xs, eq, es[:1], off), (ex, xq, xs, eq[:0], es[:0], off[:1]),
        (F.quantize_f8, x.cpu()), (F.quantize_f8, x[0]), (F.quantize_f8, x.long()), (F.quantize_f8, x.double()), (F.quantize_f8, x[:, :0]),
        (srt, ids.cpu(), 4), (srt, ids[0], 4), (srt, ids.float(), 4), (srt, ids, 0), (srt, ids, 4097), (srt, ids, "4"), (srt, ids[:, :0], 4),
        (rws, x.cpu(), tok), (rws, x, tok.cpu()), (rws, x, tok.long()), (rws, x, tok[:, None]), (rws, x.double(), tok), (rws, x[0], tok), (rws, x[:, :0], tok),
        (cmb, x.cpu(), slots), (cmb, x, slots.cpu()), (cmb, x, slots.long()), (cmb, x, slots[0]), (cmb, x, slots[:, :0]), (cmb, x.long(), slots),
        (cmb, x, slots, w[:2]), (cmb, x, slots, w.cpu()), (cmb, x, slots, w.double()), (cmb, x[:, :0], slots),
        (grd, x[:3], x, slots, w, tok[:5]), (grd, x[:2], x, slots, w, tok), (grd, x[:3].half(), x, slots, w, tok), (grd, x[:3, :63], x, slots, w, tok),
        (grd, x[:3], x, slots, w[:2], tok), (grd, x[:3], x, slots, w.cpu(), tok), (grd, x[:3].cpu(), x, slots, w, tok), (grd, x[:3], x, slots, w, tok.long()),
        (grd, x[:3], x, slots.long(), w, tok), (grd, x[:3], x, slots, None, tok),
        (grd, x[:1], x, torch.zeros((1, 129), dtype=torch.int32, device="cuda"), torch.ones((1, 129), device="cuda"), tok),
        (grd, torch.ones((3, 32769), device="cuda"), torch.ones((6, 32769), device="cuda"), slots, w, tok)]
    for i, (call, *args) in enumerate(bad):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            call(*args)
            print("not refused:", i, call.__name__)
    with pytest.raises((TypeError, ValueError)):
        lin(xq, xs, wq, ws, out_dtype=torch.int8)
    for call in (F.quantize_q8, ):
        with pytest.raises((TypeError, ValueError)):
            call(x, "e4m3_g64")
    # nothing that was refused left an error behind
    assert torch.equal(lin(xq, xs, wq, ws, out_dtype=torch.float32), exact_product(xq, xs, wq, ws).float())


def test_empty_calls(F):
    """No rows, no pairs, no experts' weights to read: empty results, or zeros where there is a row."""
    xq, xs, wq, ws = expert_operands(0, 3, 130, 200, 0)
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert F.f8_linear_experts(xq, xs, wq, ws, off).shape == (0, 130) and F.f8_linear_experts(xq, xs, wq, ws, off, none).shape == (0, 130)
    offsets, tokens, slots = F.expert_sort(torch.empty((0, 4), dtype=torch.int64, device="cuda"), 3)
    assert offsets.tolist() == [0, 0, 0, 0] and tokens.shape == (0,) and slots.shape == (0, 4)
    x = torch.ones((0, 8), device="cuda")
    assert F.expert_rows(x, none).shape == (0, 8) and torch.equal(F.expert_rows(x, off), torch.zeros((4, 8), device="cuda"))
    slots = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    w = torch.full((3, 2), float("nan"), device="cuda")
    assert torch.equal(F.expert_combine(x, slots, w), torch.zeros((3, 8), device="cuda"))
    dy, dw = F.expert_combine_grad(torch.ones((3, 8), device="cuda"), x, slots, w, none)
    assert dy.shape == (0, 8) and torch.equal(dw, torch.zeros((3, 2), device="cuda"))
    q, s = F.quantize_f8(torch.ones((0, 8), device="cuda"))
    assert q.shape == (0, 8) and s.shape == (0, 1)


@pytest.mark.parametrize("t,k", [(30, 8), (40, 8), (128, 8), (129, 8), (1025, 4)])
def test_sort_of_the_most_experts(F, t, k):
    """4096 counts per wave, where those of four waves are 64 KB of LDS and of eight 128."""
    ids = route(t, k, 4096, t, drop=0.1)
    for got, want in zip(F.expert_sort(ids, 4096), o.sort(ids.cpu().numpy(), 4096)):
        assert (got.cpu().numpy() == want).all()


@pytest.mark.parametrize("t,k,experts", [(700, 8, 60), (9000, 8, 512), (1100, 2, 4096)])
def test_captured_sort(F, t, k, experts):
    """Two captured sorts of several workgroups, each with a workspace of its own, replayed with eager sorts between."""
    a, b = route(t, k, experts, 0), route(t, k, experts, 1)
    F.expert_sort(a, experts)
    graphs, outs = [], []
    for ids in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(F.expert_sort(ids, experts))
        graphs.append(graph)
    for seed in range(3):
        a.copy_(route(t, k, experts, 2 + seed, drop=0.1))
        b.copy_(route(t, k, experts, 9 + seed))
        graphs[0].replay()
        eager = F.expert_sort(b, experts)
        graphs[1].replay()
        torch.cuda.synchronize()
        for got, want in zip(outs[1], eager):
            assert torch.equal(got, want)
        for got, want in zip(outs[0], F.expert_sort(a, experts)):
            assert torch.equal(got, want)


def test_two_streams_at_once(F):
    """Sorts, products and sums of two batches, enqueued on two streams without a wait between them."""
    t, k, experts, h = 2000, 6, 32, 640
    wq, ws = F.quantize_f8(torch.randn((experts, 384, h), device="cuda"))
    batch = [(route(t, k, experts, i), *F.quantize_q8(torch.randn((t, h), device="cuda"), FMT), torch.rand((t, k), device="cuda")) for i in (0, 1)]

    def run(ids, q, s, w):
        offsets, tokens, slots = F.expert_sort(ids, experts)
        y = F.f8_linear_experts(q, s, wq, ws, offsets, tokens)
        return F.expert_combine(y, slots, w), *F.expert_combine_grad(torch.ones_like(y[:t]), y, slots, w, tokens)
    want = [run(*b) for b in batch]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for i in (0, 1):
            with torch.cuda.stream(side[i]):
                got[i].append(run(*batch[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for run_ in got[i]:
            assert all(torch.equal(g, e) for g, e in zip(run_, want[i]))


def test_rows_past_2_31(F):
    """Strides that take rows past 2^31 and 2^32 elements: their values are those of the same rows side by side."""
    h, stride, n = 256, (1 << 28) + 64, 18           # 18 rows over 4.8e9 bf16 elements
    big = torch.empty(n * stride, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(big, (n, h), (stride, 1))
    x.copy_(torch.randn((n, h), device="cuda"))
    small = x.clone().contiguous()
    tokens = torch.tensor([17, 3, -1, 9, 16, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(F.expert_rows(x, tokens), F.expert_rows(small, tokens))
    slots = torch.tensor([[17, 0], [16, -1], [9, 8]], dtype=torch.int32, device="cuda")
    w = torch.rand((3, 2), device="cuda")
    assert torch.equal(F.expert_combine(x, slots, w), F.expert_combine(small, slots, w))
    tok = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    for t, row in enumerate(slots.tolist()):
        tok[[r for r in row if r >= 0]] = t
    for got, want in zip(F.expert_combine_grad(small[:3], x, slots, w, tok), F.expert_combine_grad(small[:3], small, slots, w, tok)):
        assert torch.equal(got, want)
    for got, want in zip(F.quantize_q8(x, FMT), F.quantize_q8(small, FMT)):
        assert torch.equal(got.float(), want.float())   # (codes have no NaN)
    for got, want in zip(F.quantize_f8(x), F.quantize_f8(small)):
        assert torch.equal(got.float(), want.float())   # (codes have no NaN)


def test_outputs_and_weights_past_2_32_bytes(F):
    """Outputs of 4.3 GB and weights whose last expert begins past 2^32 bytes."""
    m, n = 17000, 131072
    xq, xs, wq, ws = exact_operands(256, 512, 128, 3)
    want = exact_product(xq, xs, wq, ws).float().bfloat16()
    rows_ = torch.arange(m, device="cuda") % 256
    bx, bs = xq.view(torch.uint8)[rows_].view(xq.dtype), xs[rows_]
    bw, bws = wq.view(torch.uint8).repeat(n // 512, 1).view(wq.dtype), ws.repeat(n // 512, 1)
    out = F.f8_linear(bx, bs, bw, bws)
    for r in (0, 8191, 16383, 16384, m - 1):
        assert torch.equal(out[r].view(-1, 512), want[r % 256].expand(n // 512, -1))
    assert torch.equal(out[:, -512:], want[rows_])
    del out
    e = 66
    big = torch.empty((e, 131072, 512), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.ones((e, 1024, 4), device="cuda")
    aq, as_, cq, cs = exact_operands(64, 131072, 512, 4)
    big[e - 1].view(torch.uint8).copy_(cq.view(torch.uint8))
    scale[e - 1] = cs
    off = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    off[e] = 64
    got = F.f8_linear_experts(aq, as_, big, scale, off, out_dtype=torch.float32)
    assert torch.equal(got, F.f8_linear(aq, as_, cq, cs, out_dtype=torch.float32))


def test_codes_that_are_copied(F):
    """Rows, and weights of experts, that do not start on 16 bytes, or whose last row cannot be read to 16 bytes."""
    xq, xs, wq, ws = expert_operands(90, 3, 70, 300, 9)
    offsets, tokens, _ = F.expert_sort(route(90, 2, 3, 1), 3)
    want = plain_experts(xq, xs, wq, ws, offsets, tokens).float()

    def off(q, by):                                  # the same codes, side by side, `by` bytes into a buffer
        b = torch.empty(q.numel() + by, dtype=torch.uint8, device="cuda")[by:].view(q.shape)
        b.copy_(q.view(torch.uint8))
        return b.view(q.dtype)
    for x, w in ((xq.contiguous(), wq), (xq, wq.contiguous()), (off(xq, 5), off(wq, 3)), (off(xq, 16), off(wq, 16))):
        assert torch.equal(F.f8_linear_experts(x, xs, w, ws, offsets, tokens, out_dtype=torch.float32), want)


def test_a_weight_that_repeats(F):
    """One weight for all experts, expanded: its rows have a stride of 0 between experts."""
    xq, xs, wq, ws = expert_operands(300, 1, 200, 256, 4)
    offsets, tokens, _ = F.expert_sort(route(100, 3, 5, 0), 5)
    e5, s5 = wq.expand(5, -1, -1), ws.expand(5, -1, -1)
    want = plain_experts(xq, xs, e5, s5, offsets, tokens)
    assert torch.equal(F.f8_linear_experts(xq, xs, e5, s5, offsets, tokens, out_dtype=torch.float32), want.float())


def test_the_same_token_twice(F):
    """A token whose ids name an expert twice has two rows there, both added; slots that repeat are added twice."""
    ids = torch.tensor([[2, 2, 0], [1, 1, 1]], device="cuda")
    offsets, tokens, slots = F.expert_sort(ids, 3)
    assert offsets.tolist() == [0, 1, 4, 6] and tokens.tolist() == [0, 1, 1, 1, 0, 0] and slots.tolist() == [[4, 5, 0], [1, 2, 3]]
    x = torch.randn((2, 40), device="cuda")
    assert torch.equal(F.expert_combine(F.expert_rows(x, tokens), slots), (x + x) + x)
    same = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    assert torch.equal(F.expert_combine(x, same), ((x[:1] + x[:1]) + x[:1]).expand(2, -1))


@pytest.fixture(scope="module")
def example(gpu):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "experts_f8.py")
    spec = importlib.util.spec_from_file_location("experts_f8", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("tokens", [1, 90])
def test_example_runs(example, tokens):
    """examples/experts_f8.py against the block in fp32.  A code is off by at most 2^-4 of its value and its square
    averages to about 2^-10.7 of the value's (uniform over the steps of an octave: 2.4%), on both sides of each product
    (3.4%), twice for the gate times the up half (4.8%), and again for down (3.4%): 6%; twice that holds for every row."""
    assert example.main(tokens, picks=3, hidden=512, inner=256, experts=6) < 0.12


def test_example_gradients(F, example):
    """Rows and Combine of the example, chained, against plain expressions in fp64: sums of k and of h products in fp32,
    each at most 2^-24 off relative to the sum of their magnitudes, and one rounding of each value stored between."""
    t, k, h, experts = 50, 3, 200, 7
    ids = route(t, k, experts, 3, drop=0.2)
    _, tokens, slots = F.expert_sort(ids, experts)
    leaf = [torch.randn((t, h), device="cuda").requires_grad_(), torch.rand((t, k), device="cuda").requires_grad_()]
    scale, d = torch.randn((t * k, h), device="cuda"), torch.randn((t, h), device="cuda")
    example.Combine.apply(example.Rows.apply(leaf[0], tokens, slots) * scale, slots, tokens, leaf[1]).backward(d)

    x, w, d64, s64 = (v.detach().double() for v in (*leaf, d, scale))
    has = (slots >= 0)[..., None]
    f = torch.where(has, s64[slots.clamp_min(0).long()], 0.0)              # [t, k, h]
    dx, dw = (w[..., None] * f * d64[:, None]).sum(1), (f * x[:, None] * d64[:, None]).sum(2)
    for got, want, size, n in ((leaf[0].grad, dx, (w[..., None] * f * d64[:, None]).abs().sum(1), k + 3),
                               (leaf[1].grad, dw, (f * x[:, None] * d64[:, None]).abs().sum(2), h + 3)):
        assert ((got.double() - want).abs() <= 1.01 * n * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("t,k,experts", [(1 << 20, 1, 512), ((1 << 20) + 77, 1, 512), (300000, 7, 4096), (1000003, 4, 3)])
def test_sort_of_several_rounds(F, t, k, experts):
    """More pairs than the workgroups' waves count at 256 each: every wave takes several rounds."""
    g = torch.Generator(device="cuda").manual_seed(k)
    ids = torch.randint(-1, experts + 1, (t, k), generator=g, device="cuda")
    offsets, tokens, slots = F.expert_sort(ids, experts)
    flat = torch.where((ids < 0) | (ids >= experts), experts, ids).reshape(-1)
    key, order = torch.sort(flat, stable=True)
    n = int((key < experts).sum())
    assert torch.equal(offsets.long(), torch.searchsorted(key, torch.arange(experts + 1, device="cuda")))
    assert torch.equal(tokens[:n].long(), order[:n] // k) and (tokens[n:] == -1).all()
    want = torch.full_like(flat, -1)
    want[order[:n]] = torch.arange(n, device="cuda")
    assert torch.equal(slots.reshape(-1).long(), want)


def test_past_the_grids(F):
    """More rows, pairs and blocks than a launch has workgroups: the ends of what the loops over them reach."""
    for m, h in ((67108869, 16), (4194309, 264), (1048579, 1032)):
        x = torch.zeros((m, h), dtype=torch.bfloat16, device="cuda")
        x[-9:] = torch.randn((9, h), device="cuda")
        q, s = F.quantize_q8(x, FMT)
        q9, s9 = F.quantize_q8(x[-9:].clone(), FMT)
        assert torch.equal(q[-9:].float(), q9.float()) and torch.equal(s[-9:], s9)
        assert torch.equal(s[:-9].amax(), s[0, 0]) and not q[:64].float().any()
        del x, q, s
    w = torch.randn((1048580, 1, 8), device="cuda")
    q, s = F.quantize_f8(w)
    q9, s9 = F.quantize_f8(w[-9:].clone())
    assert torch.equal(q[-9:].float(), q9.float()) and torch.equal(s[-9:], s9)
    p = 4194309
    y = torch.randn((p, 8), device="cuda")
    at = torch.randperm(p, device="cuda").int()
    assert torch.equal(F.expert_combine(y, at[:, None]), y[at.long()])
    assert torch.equal(F.expert_rows(y, at), y[at.long()])
    at = torch.randint(0, 1 << 20, (8388700,), device="cuda", dtype=torch.int32)
    assert torch.equal(F.expert_rows(y[:1 << 20], at), y[at.long()])


def test_the_most_rows(F):
    """2^24 rows: the tallest product."""
    xq, xs, wq, ws = exact_operands(256, 16, 16, 1)
    rows_ = torch.arange(1 << 24, device="cuda") % 256
    bx = xq.view(torch.uint8)[rows_].view(xq.dtype)
    out = F.f8_linear(bx, xs[rows_], wq, ws)
    want = exact_product(xq, xs, wq, ws).float().bfloat16()
    assert torch.equal(out.view(-1, 256, 16), want.expand(1 << 16, -1, -1))


@pytest.mark.parametrize("t,k,h,dt", [(4001, 8, 2560, torch.bfloat16), (3000, 6, 2571, torch.float32), (9000, 4, 1000, torch.float16),
                                      (70000, 3, 255, torch.uint8), (2500, 8, 1500, torch.bfloat16), (5000, 2, 4097, torch.bfloat16),
                                      (9, 900, 4199, torch.int8), (2100, 4, 1030, torch.int32), (4000000, 5, 3, torch.bfloat16)])
def test_large_rows(F, t, k, h, dt):
    """Rows of tokens that share them, more than the L2 holds: every length of a part, rows that start anywhere, a third without a token."""
    assert t * k * h * dt.itemsize > 32 << 20
    g = torch.Generator(device="cuda").manual_seed(h)
    bits = torch.randint(0, 256, (t * (h + 1) * dt.itemsize,), generator=g, device="cuda", dtype=torch.uint8)
    x = bits.view(dt).view(t, h + 1)[:, 1:]
    tokens = torch.randint(-t // 2, t, (t * k,), generator=g, device="cuda", dtype=torch.int32)
    tokens[5::7] = t                                 # (behind the last)
    got = F.expert_rows(x, tokens)
    one = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[dt.itemsize]
    x, got = x.contiguous().view(one), got.view(one)
    for part in range(0, t * k, 1 << 22):
        tk = tokens[part:part + (1 << 22)].long()
        has = ((tk >= 0) & (tk < t))[:, None]
        assert torch.equal(got[part:part + (1 << 22)], torch.where(has, x[tk.clamp(0, t - 1)], torch.zeros((), dtype=one, device="cuda")))


@pytest.mark.parametrize("t,k,h,dt", [(4001, 8, 1290, torch.bfloat16), (9000, 2, 1001, torch.float32), (3000, 4, 3333, torch.float16),
                                      (900, 3, 17000, torch.bfloat16)])
def test_large_sums_and_gradients(F, t, k, h, dt):
    """More rows than the L2 holds, some pairs dropped: against fp64, each sum's terms and its rounding off by half a step at most."""
    assert t * k * h * dt.itemsize > 32 << 20
    ids = route(t, k, 24, h, drop=0.1)
    _, tokens, slots = F.expert_sort(ids, 24)
    y, d, w = torch.randn((t * k, h), device="cuda").to(dt), torch.randn((t, h), device="cuda").to(dt), torch.rand((t, k), device="cuda")
    out = F.expert_combine(y, slots, w)
    dy, dw = F.expert_combine_grad(d, y, slots, w, tokens)
    has, at = slots >= 0, slots.clamp_min(0).long()
    half = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0   # half of fp16's least step
    for t0 in range(0, t, 500):
        p = slice(t0, t0 + 500)
        rows_ = torch.where(has[p, :, None], y[at[p]].double(), 0.0)
        terms = rows_ * w[p, :, None].double()
        err = (k + 1) * 2.0 ** -24 * terms.abs().sum(1)
        want = terms.sum(1)
        assert ((out[p].double() - want).abs() <= err + half * (want.abs() + err) + tiny).all()
        terms = rows_ * d[p, None].double()
        assert ((dw[p].double() - terms.sum(2)).abs() <= (h + 1) * 2.0 ** -24 * terms.abs().sum(2)).all()
        # one rounding from the product, or two by way of fp32 (2^-24, then half a step of what that gives)
        want = torch.where(has[p, :, None], w[p, :, None].double() * d[p, None].double(), 0.0)
        got = torch.where(has[p, :, None], dy[at[p]].double(), 0.0)
        assert ((got - want).abs() <= (half + 2.0 ** -23) * want.abs() + tiny).all()
    n = int(has.sum())
    assert not dy[n:].any()
