"""Rows into e4m3_g128, without a GPU (tests/standin.py): in the launch that a
length takes every value has a lane, and a block of 128 lies within 16 lanes."""
import json

import pytest

import standin


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    if not standin.available():
        pytest.skip("needs g++ and libfp4x.so")
    so = standin.build(tmp_path_factory.mktemp("standin"))
    return lambda code: json.loads(standin.run(so, code))


def test_rows(route):
    """Rows per workgroup are a power of two up to 64, so for 64 and 65536 rows the grid gives the lanes of a row."""
    sizes = [(m, h) for m in (64, 65536) for h in sorted({1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, *range(100, 3000, 61), *range(1024, 32769, 512),
                                                          640, 1000, 1280, 2560, 2571, 6144, 8199, 12000, 16385, 32767, 32768})]
    got = route(f"""
rt.fp4x_test_grids.restype = ctypes.c_char_p
out = []
for M, H in {sizes!r}:
    for fn, args in ((L.fp4x_quantize_q8, (P, H, B.DT_BF16, M, H)), (L.fp4x_silu_mul_q8, (P, H, P, H, B.DT_BF16, M, H)),
                     (L.fp4x_rms_norm_q8, (P, H, B.DT_BF16, None, 0, B.DT_BF16, P, B.DT_BF16, 0.0, 1e-6, M, H))):
        tail = (None, 0, None, 0, None) if fn is L.fp4x_rms_norm_q8 else (None,)
        rc, names = launched(fn, *args, 4, P, H, P, *tail)
        assert rc == B.OK and len(names) == 1, L.fp4x_last_error()
        out.append((M, H, names[0], *map(int, rt.fp4x_test_grids().split())))
print(json.dumps(out))
""")
    seen = set()
    for m, h, name, grid, block in got:
        most, c = int(name.split("Lb1ELi")[1].split("E")[0]), int(name.split("ELi")[-1].split("E")[0])
        assert "row_q8" in name and block <= most and block * grid % m == 0, (m, h, name, grid, block)
        lanes = block * grid // m
        assert lanes * c * 8 >= h, (m, h, name, grid, block)
        assert lanes % 64 == 0 if lanes > 64 else 64 % lanes == 0      # whole waves, or several rows to one
        assert lanes % 16 == 0 or c == 1 and lanes * 8 >= h            # chunks of a block side by side
        seen.add((c, lanes <= 64))
    assert {c for c, _ in seen} == {1, 2, 3, 4, 5} and {(2, True), (3, True), (5, True)} <= seen, seen
