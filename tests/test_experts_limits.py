"""Sizes past what the kernels of experts count in 32 bits are refused before any
launch, without a GPU; the largest below are taken (tests/standin.py)."""
import pytest

import standin


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    if not standin.available():
        pytest.skip("needs g++ and libfp4x.so")
    so = standin.build(tmp_path_factory.mktemp("standin"))
    return lambda code: standin.run(so, code)


def test_combine(route):
    """A kernel steps over the picks by up to 8 and over a row's values by 512: both stay below 2^31."""
    out = route("""
most = (1 << 31) - 512
for k, H in ((8, most), (most, 8), (most, most), (1, 1)):
    rc, names = launched(L.fp4x_expert_combine, P, H, B.DT_BF16, 24, P, P, B.DT_F32, P, H, 1, k, H, None)
    assert rc == B.OK and len(names) == 1, (k, H, L.fp4x_last_error())
for k, H in ((8, most + 1), (most + 1, 8), (8, (1 << 31) - 1), ((1 << 31) - 1, 8)):
    for T in (1, 5):
        for w in (P, None):
            rc, names = launched(L.fp4x_expert_combine, P, H, B.DT_BF16, 24, P, w, B.DT_F32, P, H, T, k, H, None)
            assert rc == B.ERR_ARG and not names and L.fp4x_last_error().startswith(b"expert_combine:"), (k, H)
print("ok")
""")
    assert out.strip() == "ok"
