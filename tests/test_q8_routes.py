"""What the 8-bit activation path launches, without a GPU (tests/standin.py, 256
CUs): the kernel that a size takes and its grid."""
import json
import math
import re

import pytest

import standin


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    if not standin.available():
        pytest.skip("needs g++ and libfp4x.so")
    so = standin.build(tmp_path_factory.mktemp("standin"))
    return lambda code: json.loads(standin.run(so, code))


HEAD = """
rt.fp4x_test_grids.restype = ctypes.c_char_p


def one(fn, *args):
    rc, names = launched(fn, *args)
    assert rc == B.OK and len(names) == 1, (rc, names, args)
    grid, block = map(int, rt.fp4x_test_grids().split())
    return names[0], grid, block
"""


def test_products(route):
    sizes = [(m, n, k) for m in (1, 17, 40, 64, 100, 250, 512, 1100, 2851, 4096, 70000) for n in (1, 64, 2560, 18470)
             for k in (1, 100, 128, 129, 199, 256, 300, 384, 385, 512, 520, 640, 2560, 10240)]
    got = route(HEAD + f"""
out = []
for M, N, K in {sizes!r}:
    ld = K + 15 & -16
    out.append(one(L.fp4x_w8a8_linear, P, ld, P, P, ld, P, None, P, N, B.DT_BF16, M, N, K, None))
print(json.dumps(out))
""")
    several, kernels = 0, set()
    for (m, n, k), (name, grid, block) in zip(sizes, got):
        v = [int(x) for x in re.findall(r"L[ib](\d+)E", name)]
        kts = math.ceil(k / 128)
        if "i8_ring" in name:
            mt, nt, w, _ = v
            assert block == 64 * w and grid == math.ceil(m / (16 * mt)) * math.ceil(n / (16 * nt)), (m, n, k)
        else:
            assert "i8_tile" in name
            bm, bn, wm, wn, stages, tail = v
            tiles = math.ceil(m / bm) * math.ceil(n / bn)
            assert block == 64 * wm * wn and grid <= tiles and tail == (k % 128 != 0), (m, n, k)
            if grid < tiles:                         # several tiles per workgroup: scales of at most two tiles at a time
                several += 1
                assert kts > stages, (m, n, k, name, grid)
        kernels.add(name)
    assert several > 20 and len(kernels) > 11        # forms, with and without a K that ends inside a k-tile


def test_rows(route):
    sizes = [(m, h) for m in (1, 300, 777, 5000) for h in (1, 8, 31, 256, 257, 640, 2560, 2571, 6144, 8192, 8193, 12000,
                                                           16385, 32768)]
    got = route(HEAD + f"""
out = []
for M, H in {sizes!r}:
    out.append(one(L.fp4x_quantize_q8, P, H, B.DT_BF16, M, H, 0, P, H, P, None))
print(json.dumps(out))
""")
    for (m, h), (name, grid, block) in zip(sizes, got):
        chunks = int(re.findall(r"Li(\d+)E", name)[-1])
        assert "row_q8" in name and block <= 1024
        if h <= 256:                                 # rows share a workgroup
            lanes = max(4, 1 << (math.ceil(h / 8) - 1).bit_length())
            assert chunks == 1 and block == 256 and grid == math.ceil(m * lanes / 256), (m, h)
        elif h <= 512 * chunks:                      # a wave per row
            assert block == 256 and grid == math.ceil(m / 4), (m, h)
        else:
            assert grid == m and 8 * chunks * (block - 64) < h <= 8 * chunks * block, (m, h, name, block)
