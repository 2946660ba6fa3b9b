"""Experts on the GPU at sizes next to a limit of their launches."""
import numpy as np
import pytest
import torch

from oracle import f8 as o
from test_gpu_experts import close, route

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F(gpu):
    import fp4x_kernels
    return fp4x_kernels


@pytest.mark.parametrize("t,k,experts", [(350, 2, 4092), (350, 2, 4093), (350, 2, 4095), (4500, 2, 2046), (4500, 2, 2047), (4500, 2, 2048),
                                         (1500, 2, 1023), (1500, 2, 1024)])
def test_sorts_next_to_64_kb_of_lds(F, t, k, experts):
    """Counts of 4, 8 and 16 waves that fill 64 KB of LDS with the waves' totals, or pass it by those alone."""
    ids = route(t, k, experts, experts, drop=0.1)
    want = o.sort(ids.numpy(), experts)
    for got, w in zip(F.expert_sort(ids.cuda(), experts), want):
        assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.parametrize("t,k,experts,h", [(1, 1, 3, 5), (3, 8, 512, 2560), (70, 3, 7, 9), (333, 6, 60, 131), (40, 128, 200, 16), (2100, 8, 24, 1288)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_gradient_of_pairs_taken_out_after_the_sort(F, t, k, experts, h, dt):
    """Slots set to -1 behind expert_sort (an expert's capacity is full): their rows keep their token and get zeros, through
    the C entry, whose dy is the caller's and holds something else before."""
    import _fp4x as B
    g = torch.Generator().manual_seed(h)
    _, tokens, slots = F.expert_sort(route(t, k, experts, t, drop=0.2).cuda(), experts)
    full = (torch.rand((t, k), generator=g) < 0.3).cuda()
    full[0, 0] = True
    slots = torch.where(full, -1, slots)
    y, d, w = torch.randn((t * k, h), generator=g).to(dt).cuda(), torch.randn((t, h), generator=g).to(dt).cuda(), torch.rand((t, k), generator=g).cuda()
    dy, dw = torch.full((t * k, h), 7.0, dtype=dt, device="cuda"), torch.full((t, k), 7.0, device="cuda")
    code = B.DT_F32 if dt == torch.float32 else B.DT_BF16
    B.check(B.lib().fp4x_expert_combine_grad(d.data_ptr(), h, y.data_ptr(), h, code, t * k, slots.data_ptr(), tokens.data_ptr(), w.data_ptr(), B.DT_F32,
                                             dy.data_ptr(), h, dw.data_ptr(), t, k, h, B.stream_of(y)), "expert_combine_grad")
    want, dwant, bound = o.combine_grad(d.double().cpu().numpy(), y.double().cpu().numpy(), slots.cpu().numpy(), w.double().cpu().numpy())
    close(dy, want, np.abs(want) * 2.0 ** -24)
    close(dw, dwant, bound)
    none = torch.ones(t * k, dtype=torch.bool, device="cuda")
    none[slots[slots >= 0].long()] = False
    assert none.any() and not dy[none].any() and not dw[slots < 0].any()
    for got, same in zip(F.expert_combine_grad(d, y, slots, w, tokens), (dy, dw)):
        assert torch.equal(got, same)
