"""What f8_linear, f8_linear_experts, expert_sort and the rows of e4m3_g128
launch, without a GPU (tests/standin.py, 256 CUs): the kernel and grid that a size
takes, and that the GPU tests' sizes cover every kind of launch."""
import json
import math

import pytest

import standin
from test_gpu_f8_forms import DENSE, EXPERTS


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    if not standin.available():
        pytest.skip("needs g++ and libfp4x.so")
    so = standin.build(tmp_path_factory.mktemp("standin"))
    return lambda code: json.loads(standin.run(so, code))


HEAD = r"""
import math, random, re
rt.fp4x_test_grids.restype = ctypes.c_char_p
OUT = (B.DT_BF16, B.DT_F32)


def shape(name):
    # tile height and width, whether a ring
    v = [int(x) for x in re.findall(r"L[ib](\d+)E", name)]
    return (16 * v[0], 16 * v[1], True) if "f8_ring" in name else (v[0], v[1], False)


def dense(M, N, K, b16):
    ld = K + 15 & -16
    rc, names = launched(L.fp4x_f8_linear, P, ld, P, 1, M, P, ld, P, None, P, N, OUT[b16], M, N, K, None)
    assert rc == B.OK and len(names) == 1, L.fp4x_last_error()
    grid, block = map(int, rt.fp4x_test_grids().split())
    bm, bn, ring = shape(names[0])
    tiles = math.ceil(M / bm) * math.ceil(N / bn)
    assert names[0].endswith(f"Lb0ELb{b16}EEEvNS_6F8ArgsE"), names[0]
    return [L.fp4x_f8_form(M, N, K, OUT[b16]), K % 128 == 0, grid < tiles, grid, tiles, bm, bn, ring, block, names[0]]


def experts(M, N, K, E, b16):
    ld = K + 15 & -16
    rc, names = launched(L.fp4x_f8_linear_experts, P, ld, P, 1, M, M, None, P, E, P, ld, N * ld, P, P, N, OUT[b16], M, N, K, None)
    assert rc == B.OK and len(names) == 1, L.fp4x_last_error()
    grid, block = map(int, rt.fp4x_test_grids().split())
    bm, bn, ring = shape(names[0])
    hit = min(M, E)
    tiles = ((M - hit) // bm + hit) * math.ceil(N / bn)
    assert names[0].endswith(f"Lb1ELb{b16}EEEvNS_6F8ArgsE"), names[0]
    return [L.fp4x_f8_experts_form(M, N, K, E, OUT[b16]), K % 128 == 0, grid < tiles, grid, tiles, bm, bn, ring, block, names[0]]


rng = random.Random(5)
log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
"""

SHAPES = [(16, 16), (16, 32), (32, 32), (32, 64), (64, 64), (64, 128), (128, 128), (128, 128), (256, 128), (256, 256)]


def drawn(route, call, sizes):
    return route(HEAD + f"""
out = []
for i in range(12000):
    b = i & 1
    K = log(16, 6000)
    if i & 2:
        K = 128 * max(1, K // 128)
    out.append((b, {call}))
print(json.dumps(out))
""")


def test_products(route):
    got = drawn(route, "dense(log(1, 9000), log(16, 20000), K, b)", None)
    for b, (form, whole, several, grid, tiles, bm, bn, ring, block, name) in got:
        assert (bm, bn) == SHAPES[form] and ring == (form < 4) and block in (256, 512)
        assert grid <= tiles and (grid == tiles or not ring)
        # several tiles per workgroup: the bias of at most two tiles at a time
        if several:
            assert grid in (256, 512)
    kinds = {(b, *v[:3]) for b, v in got}
    ran = {(b, *v[:3]) for b in (0, 1) for v in route(HEAD + f"print(json.dumps([dense(*s, {b}) for s in {DENSE[b]!r}]))")}
    # the long draw finds a few kinds that only sizes too large for a test reach
    assert len(kinds - ran) == 0, sorted(kinds - ran)
    assert {(0, f) for f in range(10)} | {(1, f) for f in (0, 1, 2, 4, 5, 7)} == {k[:2] for k in ran}


def test_experts(route):
    got = drawn(route, "experts(log(1, 20000), log(16, 3000), K if K < 3000 else K // 2, log(1, 600), b)", None)
    for b, (form, whole, several, grid, tiles, bm, bn, ring, block, name) in got:
        assert (bm, bn) == SHAPES[form] and ring == (form < 4)
        assert grid % 8 == 0 and (grid >= tiles if ring else grid * 34 >= tiles)   # lane j of 64 holds tile j
    kinds = {(b, *v[:3]) for b, v in got}
    ran = {(b, *v[:3]) for b in (0, 1) for v in route(HEAD + f"print(json.dumps([experts(*s, {b}) for s in {EXPERTS[b]!r}]))")}
    assert len(kinds - ran) == 0, sorted(kinds - ran)
    assert {(0, f) for f in (1, 2, 4, 5, 7, 9)} | {(1, f) for f in (1, 2, 4, 5, 7)} == {k[:2] for k in ran}


def test_expert_tiles_fit_the_lanes(route):
    """Grids of few slots and many tiles: a workgroup's share of the most tiles that there can be stays below 64."""
    got = route(HEAD + """
out = []
for M, N, K, E in ((1 << 20, 16384, 128, 4096), (1 << 24, 256, 16, 1), (300000, 20000, 256, 512), (1 << 22, 4096, 64, 64)):
    for b in (0, 1):
        out.append(experts(M, N, K, E, b))
print(json.dumps(out))
""")
    for form, _, _, grid, tiles, *_ in got:
        run = math.ceil(tiles / 8)                   # an XCD's, over grid / 8 workgroups
        assert math.ceil(run / (grid // 8)) <= 64, (form, grid, tiles)


def test_sorts(route):
    sizes = [(t, k, e) for t in (0, 1, 3, 32, 33, 128, 129, 512, 513, 4001, 70000, 1 << 20) for k in (1, 8) for e in (1, 60, 512, 2048, 2049, 4096)]
    got = route(HEAD + f"""
out = []
for t, k, e in {sizes!r}:
    need = L.fp4x_expert_sort_workspace(t, k, e)
    rc, names = launched(L.fp4x_expert_sort, P, 1, k, t, k, e, P, P, P, P if need else None, need, None)
    assert rc == B.OK, L.fp4x_last_error()
    out.append((names, rt.fp4x_test_grids().decode().split(), need))
    if need:
        rc, names = launched(L.fp4x_expert_sort, P, 1, k, t, k, e, P, P, P, P, need - 1, None)
        assert rc == B.ERR_ARG and not names
print(json.dumps(out))
""")
    waves = set()
    for (t, k, e), (names, grids, need) in zip(sizes, got):
        p, w = t * k, int(names[-1].split("ILi")[1].split("E")[0])
        chunks, block = int(grids[-2]), int(grids[-1])
        waves.add(w)
        assert 64 * w <= block <= 1024 and block % 64 == 0 and w * e * 4 <= 160 * 1024 - 1024
        assert "sort_place" in names[-1] and len(names) == (2 if need else 1)
        assert need == (chunks * e * 4 if chunks > 1 else 0) and chunks <= 256
        rounds = math.ceil(p / (256 * 256 * w))
        if chunks == 1:
            assert p <= 256 * w
        else:
            assert (chunks - 1) * 256 * w * rounds < p <= chunks * 256 * w * rounds
    assert waves == {1, 4, 8, 16}


def test_rows(route):
    """Rows of e4m3_g128: every value has a lane, and a block of 128 lies within 16 lanes."""
    sizes = [(m, h) for m in (1, 300, 5000, 40000) for h in (1, 8, 31, 256, 257, 512, 640, 1000, 1280, 2560, 2571, 6144, 8192, 12000, 16385, 32768)]
    got = route(HEAD + f"""
out = []
for M, H in {sizes!r}:
    rc, names = launched(L.fp4x_quantize_q8, P, H, B.DT_BF16, M, H, 4, P, H, P, None)
    assert rc == B.OK and len(names) == 1
    out.append((names[0], *map(int, rt.fp4x_test_grids().split())))
print(json.dumps(out))
""")
    seen = set()
    for (m, h), (name, grid, block) in zip(sizes, got):
        most, c = int(name.split("Lb1ELi")[1].split("E")[0]), int(name.split("ELi")[-1].split("E")[0])
        assert "row_q8" in name and block <= most
        rows = math.ceil(m / grid)                   # per workgroup, where it has several
        lanes = block // rows if block == 256 and grid < m else block
        assert lanes * c * 8 >= h or lanes >= 4 and block == 256, (m, h, name, block, grid)
        seen.add(c)
    assert seen == {1, 2, 3, 4, 5}
