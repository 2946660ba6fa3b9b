"""rms_norm_q8: which residual outputs may share memory with an input, without a
GPU (tests/standin.py): the input's own rows in place, and rows that lie between
them; anything else would be read by one workgroup while another writes it."""
import json
import random

import pytest

import standin

H = 64


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    if not standin.available():
        pytest.skip("needs g++ and libfp4x.so")
    so = standin.build(tmp_path_factory.mktemp("standin"))
    return lambda calls: json.loads(standin.run(so, HEAD + f"print(json.dumps([norm(**c) for c in {calls!r}]))"))


# addresses and strides are counted in elements of each tensor's own type, from one base
HEAD = f"""
H = {H}
FAR = 1 << 30


def norm(x=FAR, xs=H, r=2 * FAR, rs=H, out=3 * FAR, os=H, w=4 * FAR, M=8, rdt=B.DT_BF16, wdt=B.DT_BF16):
    size = dict([(B.DT_BF16, 2), (B.DT_F32, 4)])
    at = lambda e, dt: ctypes.c_void_p((1 << 40) + e * size[dt])
    rc, names = launched(L.fp4x_rms_norm_q8, at(x, B.DT_BF16), xs, B.DT_BF16, at(r, rdt), rs, rdt, at(w, wdt), wdt, 0.0,
                         1e-6, M, H, 0, ctypes.c_void_p(1 << 50), H, ctypes.c_void_p(1 << 51), at(out, rdt), os, None, 0,
                         None)
    assert (rc == B.ERR_ARG) == (not names) and rc in (B.OK, B.ERR_ARG)
    return rc == B.OK
"""


def test_overlaps(route):
    wide = 2 * H
    good = [dict(),
            dict(out=0, r=0),                                            # over the residual
            dict(out=0, x=0),                                            # over x
            dict(out=0, r=0, x=0),
            dict(out=0, os=wide, r=0, rs=wide),
            dict(out=0, r=8 * H), dict(out=8 * H, r=0),                  # behind and before it
            dict(out=0, os=wide, r=H, rs=wide), dict(out=H, os=wide, r=0, rs=wide),   # the other half of wide rows
            dict(out=0, os=wide, x=H, xs=wide), dict(out=3 * wide + H, os=wide, x=0, xs=wide),
            dict(out=0, r=0, M=1, os=5, rs=9),                           # one row: its stride is not used
            dict(out=H, r=0, rs=0), dict(out=0, r=8 * H, rs=0),          # one row read by all, beside the output
            dict(out=0, os=wide, r=H, rs=4 * H), dict(out=H, os=4 * H, r=0, rs=wide),  # strides that differ, rows that do not meet
            dict(out=0, w=8 * H), dict(out=H, w=0), dict(out=0, os=wide, w=H)]
    bad = [dict(out=1, r=0), dict(out=0, r=1), dict(out=H, r=0), dict(out=0, r=H), dict(out=0, r=7 * H),
           dict(out=1, x=0), dict(out=7 * H, x=0), dict(out=0, x=7 * H + 63),
           dict(out=0, os=wide, r=H - 1, rs=wide), dict(out=H - 1, os=wide, r=0, rs=wide),
           dict(out=0, os=wide, x=wide, xs=wide), dict(out=wide, os=wide, x=1, xs=wide),
           dict(out=0, r=0, rs=0), dict(out=0, r=3 * H, rs=0), dict(out=0, x=H, xs=0),   # one row read by all
           dict(out=0, os=wide, r=0, rs=H), dict(out=0, os=H, r=0, rs=wide), dict(out=0, os=wide, r=H, rs=3 * H),
           dict(out=0, x=0, rdt=1), dict(out=0, r=0, rdt=1, x=0),        # another type's rows
           dict(out=0, w=0), dict(out=0, w=H - 1), dict(out=H - 1, w=0), dict(out=0, w=0, M=1), dict(out=0, os=wide, w=H + 1)]
    assert route(good) == [True] * len(good)
    assert route(bad) == [False] * len(bad)


def test_overlaps_drawn(route):
    """Against the elements themselves."""
    rng = random.Random(5)
    calls, want = [], []
    for _ in range(1500):
        M = rng.randint(1, 6)
        c = dict(M=M, out=rng.randint(0, 400), os=rng.randint(H, 3 * H), r=rng.randint(0, 400), rs=rng.randint(0, 3 * H))
        if rng.random() < 0.4:
            c["rs"] = c["os"]
        if rng.random() < 0.1:
            c["r"] = c["out"]
        calls.append(c)
        a, b = ({p + i * s + k for i in range(M) for k in range(H)} for p, s in ((c["out"], c["os"]), (c["r"], c["rs"])))
        want.append(not a & b or (c["out"] == c["r"] and (M == 1 or c["os"] == c["rs"])))
    assert route(calls) == want and 150 < sum(want) < 1350
