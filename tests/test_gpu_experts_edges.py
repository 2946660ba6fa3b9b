"""Experts on the GPU at sizes next to a limit of their launches."""
import numpy as np
import pytest

from oracle import f8 as o
from test_gpu_experts import route

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
