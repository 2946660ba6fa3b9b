"""Every kind of launch of f8_linear and f8_linear_experts on the GPU: each form,
with a K of whole blocks and one that ends inside a block, with one and with
several tiles per workgroup.  Sums are exact in fp32 here, so results equal the
definition bit for bit (tests/test_f8_routes.py checks that the sizes lead to
these launches)."""
import pytest
import torch

from test_gpu_experts import expert_operands, plain_experts
from test_gpu_f8 import exact_operands, exact_product

pytestmark = pytest.mark.gpu

# 16-bit outputs, then fp32
DENSE = [[(2, 19, 18), (1, 16, 128), (287, 248, 17), (197, 309, 128), (354, 355, 19), (401, 300, 128), (403, 636, 3396), (710, 354, 3584),
          (648, 907, 17), (681, 785, 128), (3250, 2487, 19), (4619, 1704, 461), (5909, 1381, 128), (275, 18046, 512), (3278, 963, 17),
          (1757, 1743, 128), (4279, 2276, 16), (2899, 3017, 267), (2818, 2722, 128), (1836, 4985, 384), (2031, 2254, 20), (2379, 1697, 128),
          (5375, 2331, 147), (7858, 3727, 1844), (3664, 3443, 256), (3328, 8981, 1536)],
         [(1, 22, 16), (1, 17, 128), (273, 248, 16), (212, 293, 128), (429, 351, 17), (387, 330, 128), (1400, 406, 18), (743, 674, 128),
          (5506, 673, 640), (569, 1881, 404), (2972, 1416, 439), (1176, 906, 512), (4954, 890, 512), (2605, 1161, 141), (4328, 2593, 550),
          (1838, 1868, 256), (7433, 1335, 640)]]
EXPERTS = [[(1, 16, 18, 1), (2, 18, 128, 1), (167, 754, 23, 1), (364, 354, 128, 1), (772, 789, 24, 1), (7775, 162, 25, 64), (648, 926, 128, 1),
            (656, 2992, 128, 1), (995, 967, 16, 2), (2998, 1604, 21, 2), (889, 1245, 128, 1), (1723, 2369, 128, 1), (2891, 840, 17, 1),
            (7662, 1218, 19, 1), (860, 2333, 128, 1), (5089, 2114, 128, 1), (6593, 1838, 952, 3), (9617, 1519, 700, 6), (9644, 1326, 768, 3),
            (17671, 2534, 384, 3)],
           [(5, 19, 16, 2), (2, 16, 128, 1), (691, 269, 18, 1), (482, 291, 128, 1), (315, 1394, 18, 1), (3277, 620, 19, 2), (677, 423, 128, 1),
            (778, 2532, 128, 1), (4782, 419, 142, 2), (3466, 1486, 17, 3), (1234, 1774, 256, 1), (4079, 1312, 128, 1), (4963, 1202, 18, 1),
            (4011, 2666, 18, 2), (2745, 2372, 128, 1), (7072, 1031, 128, 3)]]
OUT = [(torch.bfloat16, torch.float16), (torch.float32,)]


@pytest.fixture(scope="module")
def F(gpu):
    import fp4x_kernels
    return fp4x_kernels


@pytest.mark.parametrize("b16,m,n,k", [(b, *s) for b in (0, 1) for s in DENSE[b]])
def test_products(F, b16, m, n, k):
    xq, xs, wq, ws = exact_operands(m, n, k, m + n)
    bias = torch.randint(-100, 101, (n,), device="cuda").float()
    want = exact_product(xq, xs, wq, ws)
    for out in OUT[b16]:
        s = xs / 64 if out == torch.float16 else xs  # within its range
        w = want / 64 if out == torch.float16 else want
        assert torch.equal(F.f8_linear(xq, s, wq, ws, out_dtype=out), w.float().to(out))
        assert torch.equal(F.f8_linear(xq, s, wq, ws, bias=bias, out_dtype=out), (w + bias.double()).float().to(out))


@pytest.mark.parametrize("b16,m,n,k,e", [(b, *s) for b in (0, 1) for s in EXPERTS[b]])
@pytest.mark.parametrize("pick", [False, True])
def test_experts(F, b16, m, n, k, e, pick):
    g = torch.Generator(device="cuda").manual_seed(m)
    size = torch.rand(e, generator=g, device="cuda") + 0.05
    ids = torch.multinomial(size, m, replacement=True, generator=g)[:, None]
    offsets, tokens, _ = F.expert_sort(ids, e)
    xq, xs, wq, ws = expert_operands(m, e, n, k, n)
    t = tokens if pick else None
    want = plain_experts(xq, xs, wq, ws, offsets, t)
    for out in OUT[b16][:1]:
        assert torch.equal(F.f8_linear_experts(xq, xs, wq, ws, offsets, t, out_dtype=out), want.float().to(out))
