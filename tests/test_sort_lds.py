"""expert_sort asks for the LDS that its kernels take beyond 64 KB, without a GPU:
a stand-in for the runtime (tests/standin.py) that keeps each launch's dynamic
LDS and what hipFuncSetAttribute allowed that kernel before it."""
import json
import re

import pytest

import standin

TOTALS = 16 * 4                                      # sort_place's wave_total[16], beside its dynamic LDS


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    if not standin.available():
        pytest.skip("needs g++ and libfp4x.so")
    text = standin.RUNTIME
    for old, new in (("int hipFuncSetAttribute(const void*, int, int) {",
                      "static std::map<const void*, int>& most() { static auto* m = new std::map<const void*, int>; return *m; }\n"
                      "static size_t cfg_lds;\n"
                      "int hipFuncSetAttribute(const void* f, int, int n) {\n  most()[f] = n;"),
                     ("(dim3_ g, dim3_ b, size_t, void*) { cfg_grid", "(dim3_ g, dim3_ b, size_t s, void*) { cfg_lds = s; cfg_grid"),
                     ("*s = 0;", "*s = cfg_lds;"),
                     ("dim3_ b, void**, size_t, void*) {", "dim3_ b, void**, size_t s, void*) {"),
                     ('std::to_string(b.x) + "\\n"', 'std::to_string(b.x) + " " + std::to_string(s) + " " + std::to_string(most()[fn]) + "\\n"')):
        assert text.count(old) == 1, old
        text = text.replace(old, new)
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(standin, "RUNTIME", text)
        so = standin.build(tmp_path_factory.mktemp("lds"))
    return lambda code: json.loads(standin.run(so, code))


# waves of a workgroup: 1, 4, 16, 8, 16; experts on both sides of what 64 KB hold of each
PAIRS = {200: 1, 700: 4, 3000: 16, 9000: 8, 1 << 19: 16}
EXPERTS = (1, 512, 1007, 1008, 1009, 1023, 1024, 1025, 2031, 2032, 2033, 2047, 2048, 2049, 4079, 4080, 4081, 4092, 4093, 4094, 4095, 4096)


def test_sorts_ask_for_their_lds(route):
    got = route(f"""
rt.fp4x_test_grids.restype = ctypes.c_char_p
out = []
for p in {list(PAIRS)!r}:
    for e in {EXPERTS!r}:
        need = L.fp4x_expert_sort_workspace(p, 1, e)
        rc, names = launched(L.fp4x_expert_sort, P, 1, 1, p, 1, e, P, P, P, P if need else None, need, None)
        assert rc == B.OK, L.fp4x_last_error()
        out.append((p, e, names, [list(map(int, g.split())) for g in rt.fp4x_test_grids().decode().splitlines()]))
print(json.dumps(out))
""")
    beyond = 0
    for p, e, names, launches in got:
        assert len(names) == len(launches) >= 1
        for name, (_, _, lds, most) in zip(names, launches):
            w = int(re.search(r"ILi(\d+)E", name).group(1))
            assert w == PAIRS[p] or e > 2048 and w == 8, (p, e, w)
            assert lds == 4 * w * e
            takes = lds + TOTALS
            if takes > 64 * 1024:
                beyond += 1
                assert most >= lds, (p, e, name, lds, most)
            assert takes <= 160 * 1024
    assert beyond > 20
