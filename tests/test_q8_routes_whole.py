"""The sizes that the GPU tests run cover every kind of launch of
w8a8_linear, without a GPU (tests/standin.py, 256 CUs): each form, with a K of
whole k-tiles and one that ends inside a k-tile, with one and with several
tiles per workgroup, as far as the choice of a form leads there at all; and the row kernels past their
largest grid."""
import json

import pytest

import standin
from test_gpu_q8 import FORM_KS, FORMS
from test_gpu_q8_edges import CAP, PAST, RAGGED, WHOLE


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    if not standin.available():
        pytest.skip("needs g++ and libfp4x.so")
    so = standin.build(tmp_path_factory.mktemp("standin"))
    return lambda code: json.loads(standin.run(so, code))


KIND = r"""
import math, random, re
rt.fp4x_test_grids.restype = ctypes.c_char_p


def kind(M, N, K):
    # form, whole k-tiles, several tiles per workgroup
    ld = K + 15 & -16
    rc, names = launched(L.fp4x_w8a8_linear, P, ld, P, P, ld, P, None, P, N, B.DT_BF16, M, N, K, None)
    assert rc == B.OK and len(names) == 1
    grid = int(rt.fp4x_test_grids().split()[0])
    v = [int(x) for x in re.findall(r"L[ib](\d+)E", names[0])]
    tile = v[:2] if "i8_tile" in names[0] else [16 * v[0], 16 * v[1]]
    tiles = math.ceil(M / tile[0]) * math.ceil(N / tile[1])
    return [L.fp4x_w8a8_form(M, N, K), K % 128 == 0, grid < tiles]
"""


def test_kinds_are_covered(route):
    sizes = WHOLE + RAGGED + [(m, n, k) for m, n in FORMS for k in FORM_KS]
    ran = {tuple(k) for k in route(KIND + f"print(json.dumps([kind(*s) for s in {sizes!r}]))")}
    drawn = {tuple(k) for k in route(KIND + """
rng = random.Random(1)
log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
out = set()
for i in range(60000):
    m, n, k = log(1, 9000), log(1, 40000), log(64, 11000)
    out.add(tuple(kind(m, n, 128 * max(1, k // 128) if i % 2 else k)))
print(json.dumps(sorted(out)))
""")}
    assert {f for f, _, _ in drawn} == set(range(11)) and any(s for _, _, s in drawn)
    assert drawn <= ran, sorted(drawn - ran)
    # what the choice does not lead to: several tiles of 64 x 64 per workgroup
    assert not any(f == 5 and several for f, _, several in drawn | ran)


def test_rows_past_the_grid(route):
    """Sizes that take a workgroup through its row loop more than once, with rows of part of a wave, of one wave and of
    several, and each number of chunks per lane that so many rows lead to."""
    got = route(KIND + f"""
out = []
for M, H in {PAST!r}:
    rc, names = launched(L.fp4x_quantize_q8, P, 8, B.DT_BF16, M, H, 0, P, H + 15 & -16, P, None)
    assert rc == B.OK and len(names) == 1
    out.append([*map(int, rt.fp4x_test_grids().split()), int(re.findall(r"Li(\\d+)E", names[0])[-1])])
print(json.dumps(out))
""")
    assert all(grid == CAP for grid, _, _ in got)
    assert [(block, chunks) for _, block, chunks in got] == [(256, 1), (256, 2), (128, 2), (128, 2), (192, 3), (832, 4)]
