"""The 8-bit activation path, as cases that can be timed: norms, gates and rows
that end in 8 bits with scales, and the product of 8-bit integers they feed.

A server that has compute to spare on its weights' bits but not on its
activations' (a prefill chunk, a batch of hundreds of sequences) multiplies
8-bit integers: the block's input is normed and quantized in one pass, every
projection is an int8 product with a scale per token and a scale per output
channel, and the gated activation of the MLP ends in 8 bits again.

A case is a dict with a "kind":

  norm    rms_norm_q8: root-mean-square norm of m rows of h values, with the
          residual's addition where `res` names its type, into `fmt`; `normed`
          asks for the unquantized rows too (a router gate reads them)
  silu    silu_mul_q8: silu(gate) * up of m rows of 2 f values into `fmt`
  quant   quantize_q8: m rows of h values into `fmt` (a weight matrix when the
          model is loaded, or an attention output before its projection)
  linear  w8a8_linear: int8 [m, k] x int8 [n, k] with both scales and a bias
          where `bias` is true, into `out`
  down    the tail of a gated MLP: silu_mul_q8 into int8, then w8a8_linear

`fmt`: int8 (codes and one fp32 scale per row), e4m3 (the same with fp8 codes),
mx8 (fp8 codes and one power of two per 32 values, as an e8m0 byte).  fp8 codes
are compared as the values they are; int8 codes have to be equal, which is why
the sum of squares is taken in 64 bits and every later step is one rounded fp32
operation: the codes are then defined to the last one.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6
_FW = None


def _fw():
    global _FW
    if _FW is None:
        pkg = os.path.join(_ROOT, "qwen3.8-flash-next-fp4-local-spark_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import fp4x_kernels
        _FW = fp4x_kernels
    return _FW


def listed():
    return [
        # a decode step's norm: one sequence with two draft rows; latency alone
        {"name": "norm_decode", "kind": "norm", "m": 3, "h": 2560, "dt": "bf16", "res": "bf16", "fmt": "int8",
         "normed": False},
        # a prefill chunk into an expert block: the router gate reads the normed rows, the linears the int8 ones
        {"name": "norm_chunk", "kind": "norm", "m": 4096, "h": 2560, "dt": "bf16", "res": "bf16", "fmt": "int8",
         "normed": True},
        # no size a multiple of anything: rows that start off every alignment
        {"name": "norm_odd_e4m3", "kind": "norm", "m": 333, "h": 2571, "dt": "f16", "res": "none", "fmt": "e4m3",
         "normed": False},
        # the gate of a dense MLP over a prefill chunk
        {"name": "silu_chunk", "kind": "silu", "m": 4096, "f": 6144, "dt": "bf16", "fmt": "e4m3"},
        # the shared expert's tail over a small prefill chunk
        {"name": "down_m512", "kind": "down", "m": 512, "n": 2560, "k": 640, "dt": "bf16", "out": "bf16"},
        # a qkv weight when the model is loaded: one scale per output channel
        {"name": "quant_weight", "kind": "quant", "m": 16384, "h": 2560, "dt": "bf16", "fmt": "int8"},
        # a ragged batch's rows, of odd length
        {"name": "quant_odd", "kind": "quant", "m": 777, "h": 6145, "dt": "f16", "fmt": "int8"},
        # one token through the shared expert's down projection: the smallest product
        {"name": "linear_m1", "kind": "linear", "m": 1, "n": 2560, "k": 640, "out": "bf16", "bias": False},
        # sixteen rows through the widest projection: the weights' bytes are the time
        {"name": "linear_m16", "kind": "linear", "m": 16, "n": 16384, "k": 2560, "out": "bf16", "bias": False},
        # 64 sequences through the attention's output projection: few columns, a long sum
        {"name": "linear_m64", "kind": "linear", "m": 64, "n": 2560, "k": 6144, "out": "f32", "bias": False},
        # a batch that fills no tile, with a bias
        {"name": "linear_m250", "kind": "linear", "m": 250, "n": 13310, "k": 2560, "out": "f16", "bias": True},
        # a prefill chunk through the widest projection: the matrix cores' case
        {"name": "linear_m4096", "kind": "linear", "m": 4096, "n": 16384, "k": 2560, "out": "bf16", "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("norm", "silu", "quant", "linear", "down"), (4, 2, 2, 6, 2))[0]
    dt = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind in ("norm", "quant"):
        fmt = rng.choice(("int8", "int8", "e4m3", "mx8"))
        h = _log(rng, 64, 12000)
        h = 32 * max(2, h // 32) if fmt == "mx8" else 16 * (h // 16) if rng.random() < 0.6 else h
        c = {"kind": kind, "m": min(_log(rng, 1, 8192), 40_000_000 // h), "h": h, "dt": dt, "fmt": fmt}
        if kind == "norm":
            c |= {"res": rng.choice(("none", dt, dt, "f32")), "normed": rng.random() < 0.3}
        return c
    if kind == "silu":
        f = _log(rng, 64, 12000)
        f = 16 * (f // 16) if rng.random() < 0.6 else f
        return {"kind": kind, "m": min(_log(rng, 1, 8192), 25_000_000 // f), "f": f, "dt": dt, "fmt": "e4m3"}
    n, k = _log(rng, 16, 18000), _log(rng, 64, 10240)
    k = 64 * max(1, k // 64) if rng.random() < 0.5 else 16 * (k // 16) if rng.random() < 0.7 else k
    m = max(1, min(_log(rng, 1, 4096), 4096 * 16384 * 2560 // (n * k)))
    c = {"kind": kind, "m": m, "n": n, "k": k, "out": rng.choice(("bf16", "bf16", "f16", "f32"))}
    return c | ({"bias": rng.random() < 0.3} if kind == "linear" else {"dt": dt})


# ------------------------------------------------------------------ inputs
def _rows(g, m, h, spread=1.0):
    """Rows of a residual stream: a size of its own for each row, and a few channels far larger than the rest."""
    size = spread * torch.exp(0.5 * torch.randn((m, 1), generator=g, device=DEV))
    channel = 1 + 15 * (torch.rand((1, h), generator=g, device=DEV) > 0.995)
    return torch.randn((m, h), generator=g, device=DEV) * size * channel


def _codes(t):
    """A float matrix as int8 rows that start on 16 bytes, with the scale of each: what a server holds."""
    m, k = t.shape
    s = t.abs().amax(-1) / 127
    q = torch.zeros((m, -(-k // 16) * 16), dtype=torch.int8, device=DEV)[:, :k]
    q.copy_((t / s[:, None]).round())
    return q, s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    s = dict(case)
    if s["kind"] in ("norm", "quant"):
        m, h = s["m"], s["h"]
        # a weight matrix when it is loaded, rows of the stream otherwise
        s["x"] = _rows(g, m, h, 0.02 if m > 8192 else 1.0).to(_DT[s["dt"]])
        if s["kind"] == "norm":
            s["w"] = (1 + 0.2 * torch.randn(h, generator=g, device=DEV)).to(_DT[s["dt"]])
            s["r"] = None if s["res"] == "none" else _rows(g, m, h, 2.0).to(_DT[s["res"]])
        return s
    if s["kind"] in ("silu", "down"):
        f = s["f"] if s["kind"] == "silu" else s["k"]
        s["gu"] = (2 * torch.randn((s["m"], 2 * f), generator=g, device=DEV)).to(_DT[s["dt"]])
    else:
        s["xq"], s["xs"] = _codes(_rows(g, s["m"], s["k"]))
        s["b"] = torch.randn(s["n"], generator=g, device=DEV) if s["bias"] else None
    if s["kind"] != "silu":
        s["wq"], s["ws"] = _codes(0.02 * torch.randn((s["n"], s["k"]), generator=g, device=DEV))
    return s


# ------------------------------------------------------------------ plain forms
def _plain_q8(v, fmt):
    """fp32 rows in 8 bits.  Divisions are by tensors: torch multiplies by a Python number's reciprocal instead."""
    m, h = v.shape
    if fmt == "mx8":
        g = v.view(m, h // 32, 32)
        e = (torch.frexp(g.abs().amax(-1, keepdim=True))[1] - 1 - 8).clamp(-127, 127)
        q = torch.ldexp(g, -e).clamp(-448, 448).to(torch.float8_e4m3fn).view(m, h)
        return q, (e.squeeze(-1) + 127).to(torch.uint8)
    top = 127.0 if fmt == "int8" else 448.0
    amax = v.abs().amax(-1, keepdim=True).clamp_min(1e-12)
    s = amax / torch.full_like(amax, top)
    y = v / s
    q = y.round().clamp(-127, 127).to(torch.int8) if fmt == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)
    return q, s.squeeze(-1)


def _plain_norm(s):
    h = s["x"].float()
    if s["r"] is not None:
        h = (h + s["r"].float()).to(s["r"].dtype)
    r = (h.double().square().mean(-1, keepdim=True) + _EPS).rsqrt().float()
    v = (h.float() * r) * s["w"].float()
    out = list(_plain_q8(v, s["fmt"]))
    if s["r"] is not None:
        out.append(h)
    if s["normed"]:
        out.append(v.to(s["x"].dtype))
    return out


def _plain_silu(gu, fmt):
    g, u = gu.float().chunk(2, -1)
    return _plain_q8(g * torch.sigmoid(g) * u, fmt)


def _plain_linear(xq, xs, wq, ws, b, out):
    y = (xq.float() @ wq.float().t()) * xs[:, None] * ws
    return (y if b is None else y + b).to(out)


def run(s):
    k = s["kind"]
    if own:
        F = _fw()
        if k == "norm":
            return F.rms_norm_q8(s["x"], s["w"], eps=_EPS, residual=s["r"], fmt=s["fmt"], normed=s["normed"])
        if k == "quant":
            return F.quantize_q8(s["x"], fmt=s["fmt"])
        if k == "silu":
            return F.silu_mul_q8(s["gu"], fmt=s["fmt"])
        if k == "linear":
            return F.w8a8_linear(s["xq"], s["xs"], s["wq"], s["ws"], bias=s["b"], out_dtype=_DT[s["out"]])
        q, sc = F.silu_mul_q8(s["gu"])
        return F.w8a8_linear(q, sc, s["wq"], s["ws"], out_dtype=_DT[s["out"]])
    if k == "norm":
        return _plain_norm(s)
    if k == "quant":
        return _plain_q8(s["x"].float(), s["fmt"])
    if k == "silu":
        return _plain_silu(s["gu"], s["fmt"])
    if k == "linear":
        return _plain_linear(s["xq"], s["xs"], s["wq"], s["ws"], s["b"], _DT[s["out"]])
    q, sc = _plain_silu(s["gu"], "int8")
    return _plain_linear(q, sc, s["wq"], s["ws"], None, _DT[s["out"]])


# ------------------------------------------------------------------ 64 bits
def _exact_codes(v, fmt):
    """(codes as the values that the format holds, scales) of 64-bit rows; int8 codes have no value of their own here."""
    if fmt == "mx8":
        m, h = v.shape
        blocks = v.reshape(m, -1, 32)
        step = torch.exp2((torch.log2(blocks.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -119)).floor() - 8))
        return (blocks / step).clamp(-448, 448).to(torch.float8_e4m3fn).double().reshape(m, h), None
    s = v.abs().amax(-1).clamp_min(1e-12) / (127 if fmt == "int8" else 448)
    return None if fmt == "int8" else (v / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).double(), s


def exact(case, seed):
    s = prepare(case, seed)
    k = s["kind"]
    if k == "norm":
        h, out = s["x"].double(), []
        if s["r"] is not None:
            out.append(h + s["r"].double())
            h = out[0].to(s["r"].dtype).double()  # the norm is that of the rows the next layer is given
        v = h * s["w"].double() / ((h * h).sum(-1, keepdim=True) / s["h"] + _EPS).sqrt()
        return [*_exact_codes(v, s["fmt"]), *out, *([v] if s["normed"] else [])]
    if k == "quant":
        return _exact_codes(s["x"].double(), s["fmt"])
    if k in ("silu", "down"):
        f = s["gu"].shape[1] // 2
        g = s["gu"][:, :f].double()
        v = g / (1 + torch.exp(-g)) * s["gu"][:, f:].double()
        if k == "silu":
            return _exact_codes(v, s["fmt"])
        xs = v.abs().amax(-1) / 127
        x, b = (v / xs[:, None]).round(), None
    else:
        x, xs, b = s["xq"].double(), s["xs"].double(), s["b"]
    y = (x * xs[:, None]) @ (s["wq"].double() * s["ws"].double()[:, None]).t()
    return y if b is None else y + b.double()


def work(case):
    c = case
    if c["kind"] in ("linear", "down"):
        m, n, k = c["m"], c["n"], c["k"]
        x = m * (k + 4) if c["kind"] == "linear" else 2 * m * k * _SIZE[c["dt"]]
        bias = 4 * n if c.get("bias") else 0
        return {"bytes": x + n * (k + 4) + bias + m * n * _SIZE[c["out"]], "flops": 2 * m * n * k}
    m, h = c["m"], c.get("h") or c["f"]
    size = _SIZE[c["dt"]]
    out = m * h + (m * h // 32 if c["fmt"] == "mx8" else 4 * m)
    if c["kind"] == "silu":
        return {"bytes": 2 * m * h * size + out, "flops": 8 * m * h}
    b = m * h * size + out
    if c["kind"] == "norm":
        b += h * size + (2 * m * h * _SIZE[c["res"]] if c["res"] != "none" else 0) + (m * h * size if c["normed"] else 0)
    return {"bytes": b, "flops": 8 * m * h}
