"""Experts in 8-bit floating point, as cases that can be timed: rows and weights
in e4m3 with a scale per block of 128, their product (dense and over the rows of
each expert), tokens sorted by expert and back, and the gradients of that.

Checkpoints in fp8 hold a scale per 128 x 128 block of a weight, and their
activations take a scale per 128 values of a row.  A block of experts in that
format runs: norm into codes, router gate, its ids sorted by expert, a product
over each expert's rows (picked by index from the tokens' codes), the gated
activation into codes, the second product, and the weighted sum of each token's
rows.  Training such a block needs the sum's gradient too.

A case is a dict with a "kind":

  quant    m rows of h values into e4m3 codes with a scale per 128: `op` is norm
           (rms_norm_q8 with the residual's addition), silu (silu_mul_q8 of m
           rows of 2 h values) or rows (quantize_q8)
  linear   f8_linear: codes [m, k] x codes [n, k], both with their scales, and a
           bias where `bias` is true, into `out`
  experts  f8_linear_experts: `tokens` rows of k values, each sent to `top` of
           `experts` experts of [n, k]; `pick` reads the rows through the sort's
           token index (the first product), else they lie sorted (the second)
  sort     expert_sort of `tokens` x `top` ids; `drop`: half of the experts are
           another rank's and their ids are negative here; `h`: the sorted rows
           of that many values too (expert_rows), 0 for none
  back     expert_combine: the weighted sum of each token's rows; with `grad` its
           gradients too, for the rows and for the weights, and the gradient of
           expert_rows, which is the same sum without weights

fp8 codes are compared as the values they are.
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
_FMT = "e4m3_g128"
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
        {"name": "norm_decode", "kind": "quant", "op": "norm", "m": 3, "h": 2560, "dt": "bf16"},
        # the experts' gated activation over a prefill chunk: 4096 tokens, 8 rows each
        {"name": "silu_sorted", "kind": "quant", "op": "silu", "m": 32768, "h": 640, "dt": "bf16"},
        # a decode step through a shared expert's down projection: the smallest product
        {"name": "linear_m3", "kind": "linear", "m": 3, "n": 2560, "k": 640, "out": "bf16", "bias": False},
        # a batch that fills no tile, a K that ends inside a block, with a bias
        {"name": "linear_odd", "kind": "linear", "m": 250, "n": 13310, "k": 2500, "out": "f16", "bias": True},
        # a prefill chunk through the widest projection: the matrix cores' case
        {"name": "linear_m4096", "kind": "linear", "m": 4096, "n": 16384, "k": 2560, "out": "bf16", "bias": False},
        # a decode step through 512 experts: gate and up projections of the few that are hit
        {"name": "experts_decode", "kind": "experts", "tokens": 3, "top": 8, "experts": 512, "n": 1280, "k": 2560,
         "pick": True, "out": "bf16"},
        # a prefill chunk through the down projections of 128 experts
        {"name": "experts_chunk", "kind": "experts", "tokens": 4096, "top": 8, "experts": 128, "n": 2560, "k": 640,
         "pick": False, "out": "bf16"},
        # a decode step's ids
        {"name": "sort_decode", "kind": "sort", "tokens": 3, "top": 8, "experts": 512, "drop": False, "h": 0, "dt": "bf16"},
        # a ragged chunk's ids on a rank that holds half of the experts, and the rows themselves (training sorts them)
        {"name": "sort_chunk", "kind": "sort", "tokens": 4001, "top": 8, "experts": 256, "drop": True, "h": 2560, "dt": "bf16"},
        # a decode step's weighted sum
        {"name": "back_decode", "kind": "back", "tokens": 3, "top": 8, "experts": 512, "h": 2560, "dt": "bf16", "grad": False},
        # rows of odd length in fp32, with the gradients: a small training batch
        {"name": "back_odd", "kind": "back", "tokens": 333, "top": 6, "experts": 60, "h": 2571, "dt": "f32", "grad": True},
        # a training step's chunk: the sum and its gradients
        {"name": "back_chunk", "kind": "back", "tokens": 4096, "top": 8, "experts": 512, "h": 2560, "dt": "bf16", "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("quant", "linear", "experts", "sort", "back"), (3, 4, 3, 2, 3))[0]
    dt = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "quant":
        h = _log(rng, 64, 12000)
        h = 64 * max(1, h // 64) if rng.random() < 0.6 else h
        return {"kind": kind, "op": rng.choice(("norm", "silu", "rows")), "m": max(1, min(_log(rng, 1, 32768), 20_000_000 // h)),
                "h": h, "dt": dt}
    if kind == "linear":
        n, k = _log(rng, 16, 18000), _log(rng, 64, 10240)
        k = 64 * max(1, k // 64) if rng.random() < 0.6 else k
        m = max(1, min(_log(rng, 1, 4096), 4096 * 16384 * 2560 // (n * k)))
        return {"kind": kind, "m": m, "n": n, "k": k, "out": rng.choice(("bf16", "bf16", "f16", "f32")),
                "bias": rng.random() < 0.3}
    experts = _log(rng, 4, 512)
    top = rng.randint(1, min(10, experts))
    if kind == "experts":
        n, k = 64 * _log(rng, 2, 40), 64 * _log(rng, 2, 40)
        if rng.random() < 0.4:
            n, k = n + rng.randint(1, 63), k + rng.randint(1, 63)
        experts = max(top, min(experts, 800_000_000 // (n * k)))
        tokens = max(1, min(_log(rng, 1, 4096), 4096 * 8 * 2560 * 1280 // (top * n * k)))
        return {"kind": kind, "tokens": tokens, "top": top, "experts": experts, "n": n, "k": k, "pick": rng.random() < 0.5,
                "out": rng.choice(("bf16", "bf16", "f16", "f32"))}
    h = _log(rng, 64, 6000)
    h = 8 * (h // 8) if rng.random() < 0.6 else h
    tokens = max(1, min(_log(rng, 1, 8192), 4096 * 8 * 2560 // (top * h)))
    if kind == "sort":
        if rng.random() < 0.5:
            h, tokens = 0, _log(rng, 1, 16384)
        return {"kind": kind, "tokens": tokens, "top": top, "experts": experts, "drop": rng.random() < 0.4, "h": h, "dt": dt}
    return {"kind": kind, "tokens": tokens, "top": top, "experts": experts, "h": h, "dt": dt, "grad": rng.random() < 0.6}


# ------------------------------------------------------------------ inputs
def _rows(g, m, h, spread=1.0):
    """Rows of a residual stream: a size of its own for each row, and a few channels far larger than the rest."""
    size = spread * torch.exp(0.5 * torch.randn((m, 1), generator=g, device=DEV))
    channel = 1 + 15 * (torch.rand((1, h), generator=g, device=DEV) > 0.995)
    return torch.randn((m, h), generator=g, device=DEV) * size * channel


def _blocks(t, b):
    """Blocks of b x 128 of the last two dimensions, padded with zeros: [.., nb, b, kb, 128]."""
    n, k = t.shape[-2:]
    t = torch.nn.functional.pad(t, (0, -k % 128, 0, -n % b))
    return t.reshape(*t.shape[:-2], -1, b, t.shape[-1] // 128, 128)


def _codes(t, b):
    """A float matrix in e4m3 with a scale per b x 128 values, as a server holds it: code rows that start on 16 bytes, an
    activation's scales (b = 1) with the rows of a block side by side."""
    n, k = t.shape[-2:]
    v = _blocks(t, b)
    s = v.abs().amax((-3, -1), keepdim=True).clamp_min(1e-12) / 448
    c = (v / s).to(torch.float8_e4m3fn).reshape(*t.shape[:-2], v.shape[-4] * b, -1)[..., :n, :k]
    q = torch.empty((*t.shape[:-1], -(-k // 16) * 16), dtype=torch.uint8, device=DEV).fill_(0x7f)[..., :k]
    q.copy_(c.view(torch.uint8))
    s = s.squeeze(-1).squeeze(-2)
    return q.view(torch.float8_e4m3fn), s if b > 1 else s.t().contiguous().t()


def _route(g, c):
    """Ids of a router: each token's `top` best experts, some of them popular; with `drop` those of another rank are -1."""
    all_ = c["experts"] * (2 if c.get("drop") else 1)
    logits = torch.randn((c["tokens"], all_), generator=g, device=DEV) + 0.5 * torch.randn(all_, generator=g, device=DEV)
    w, ids = logits.topk(c["top"], -1)
    return torch.where(ids < c["experts"], ids, torch.full_like(ids, -1)), torch.softmax(w, -1)


def _sorted(ids, experts):
    """(offsets, tokens, slots) of expert_sort."""
    t, top = ids.shape
    flat = torch.where((ids < 0) | (ids >= experts), torch.full_like(ids, experts), ids).reshape(-1)
    key, order = torch.sort(flat, stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device=ids.device)).to(torch.int32)
    kept = key < experts
    tokens = torch.where(kept, order // top, torch.full_like(order, -1)).to(torch.int32)
    slots = torch.empty_like(flat)
    slots[order] = torch.where(kept, torch.arange(t * top, device=ids.device), torch.full_like(order, -1))
    return offsets, tokens, slots.reshape(t, top).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    s, k = dict(case), case["kind"]
    dt = _DT.get(case.get("dt"))
    if k == "quant":
        m, h = s["m"], s["h"]
        if s["op"] == "silu":
            s["x"] = (2 * torch.randn((m, 2 * h), generator=g, device=DEV)).to(dt)
        else:
            s["x"] = _rows(g, m, h).to(dt)
        if s["op"] == "norm":
            s["w"] = (1 + 0.2 * torch.randn(h, generator=g, device=DEV)).to(dt)
            s["r"] = _rows(g, m, h, 2.0).to(dt)
    elif k == "linear":
        s["xq"], s["xs"] = _codes(_rows(g, s["m"], s["k"]), 1)
        s["wq"], s["ws"] = _codes(0.02 * torch.randn((s["n"], s["k"]), generator=g, device=DEV), 128)
        s["b"] = torch.randn(s["n"], generator=g, device=DEV) if s["bias"] else None
    elif k == "experts":
        s["ids"], _ = _route(g, s)
        s["offsets"], s["map"], _ = _sorted(s["ids"], s["experts"])
        s["xq"], s["xs"] = _codes(_rows(g, s["tokens"] * (1 if s["pick"] else s["top"]), s["k"]), 1)
        some = max(1, 100_000_000 // (s["n"] * s["k"]))   # experts at a time: the fp32 values need room
        parts = [_codes(0.02 * torch.randn((min(some, s["experts"] - e), s["n"], s["k"]), generator=g, device=DEV), 128)
                 for e in range(0, s["experts"], some)]
        if len(parts) == 1:
            s["wq"], s["ws"] = parts[0]
        else:
            ld = parts[0][0].stride(1)
            whole = torch.cat([p[0].view(torch.uint8).as_strided((p[0].shape[0], s["n"], ld), p[0].stride()) for p in parts])
            s["wq"], s["ws"] = whole[..., :s["k"]].view(torch.float8_e4m3fn), torch.cat([p[1] for p in parts])
    else:
        s["ids"], s["w"] = _route(g, s)
        if k == "sort":
            s["x"] = _rows(g, s["tokens"], s["h"]).to(dt) if s["h"] else None
        else:
            _, s["map"], s["slots"] = _sorted(s["ids"], s["experts"])
            s["y"] = _rows(g, s["tokens"] * s["top"], s["h"]).to(dt)
            s["dout"] = torch.randn((s["tokens"], s["h"]), generator=g, device=DEV).to(dt) if s["grad"] else None
    return s


# ------------------------------------------------------------------ plain forms
def _plain_quant(v):
    """fp32 rows in e4m3 with a scale per 128.  Divisions are by tensors: torch multiplies by a Python number's reciprocal."""
    m, h = v.shape
    b = torch.nn.functional.pad(v, (0, -h % 128)).view(m, -1, 128)
    amax = b.abs().amax(-1, keepdim=True).clamp_min(1e-12)
    s = amax / torch.full_like(amax, 448.0)
    return (b / s).clamp(-448, 448).to(torch.float8_e4m3fn).view(m, -1)[:, :h], s.squeeze(-1)


def _wide(s, k):
    """Scales per 128 columns, one per column."""
    return s.repeat_interleave(128, -1)[..., :k]


def _weight(q, s):
    n, k = q.shape[-2:]
    return q.float() * _wide(s.repeat_interleave(128, -2)[..., :n, :], k)


def _plain_experts(s):
    top, experts, n, k = s["top"], s["experts"], s["n"], s["k"]
    x = s["xq"].float() * _wide(s["xs"], k)
    if s["pick"]:
        x = x[s["map"].long()]
    rows = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(s["offsets"], rows.to(torch.int32), right=True) - 1
    if x.shape[0] <= experts:                        # few rows: each with a copy of its expert's weight
        w = _weight(s["wq"][expert], s["ws"][expert])
        return torch.bmm(w, x[:, :, None]).squeeze(-1).to(_DT[s["out"]])
    place = rows - s["offsets"][expert]              # many: each expert's rows padded to the longest
    most = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    padded = x.new_zeros((experts, most, k))
    padded[expert, place] = x
    y = torch.bmm(padded, _weight(s["wq"], s["ws"]).transpose(1, 2).contiguous())
    return y[expert, place].to(_DT[s["out"]])


def _pick(y, slots):
    """Each token's rows in fp32 [tokens, top, h], zeros where there is none."""
    rows = y.float()[slots.clamp_min(0).long()]
    return torch.where(slots[..., None] < 0, torch.zeros((), device=y.device), rows)


def _plain_back(s):
    y, slots, w, dt = s["y"], s["slots"], s["w"], s["y"].dtype
    rows = _pick(y, slots)
    out = [(rows * w[..., None]).sum(1).to(dt)]
    if s["grad"]:
        d = s["dout"].float()
        dw = (rows * d[:, None]).sum(-1)
        dy = torch.zeros_like(y)
        pairs = slots.reshape(-1).long()
        kept = (pairs >= 0).nonzero().squeeze(-1)
        dy[pairs[kept]] = (w[..., None] * d[:, None]).reshape(pairs.shape[0], -1)[kept].to(dt)
        out += [dy, dw, _pick(dy, slots).sum(1).to(dt)]
    return out


def run(s):
    k = s["kind"]
    if own:
        F = _fw()
        if k == "quant":
            if s["op"] == "norm":
                return F.rms_norm_q8(s["x"], s["w"], eps=_EPS, residual=s["r"], fmt=_FMT)
            return F.silu_mul_q8(s["x"], fmt=_FMT) if s["op"] == "silu" else F.quantize_q8(s["x"], fmt=_FMT)
        if k == "linear":
            return F.f8_linear(s["xq"], s["xs"], s["wq"], s["ws"], bias=s["b"], out_dtype=_DT[s["out"]])
        if k == "experts":
            return F.f8_linear_experts(s["xq"], s["xs"], s["wq"], s["ws"], s["offsets"],
                                       tokens=s["map"] if s["pick"] else None, out_dtype=_DT[s["out"]])
        if k == "sort":
            offsets, tokens, slots = F.expert_sort(s["ids"], s["experts"])
            return [offsets, tokens, slots] + ([F.expert_rows(s["x"], tokens)] if s["h"] else [])
        out = [F.expert_combine(s["y"], s["slots"], s["w"])]
        if s["grad"]:
            dy, dw = F.expert_combine_grad(s["dout"], s["y"], s["slots"], s["w"], s["map"])
            out += [dy, dw, F.expert_combine(dy, s["slots"])]
        return out
    if k == "quant":
        if s["op"] == "silu":
            a, b = s["x"].float().chunk(2, -1)
            return _plain_quant(a * torch.sigmoid(a) * b)
        if s["op"] == "rows":
            return _plain_quant(s["x"].float())
        h = (s["x"].float() + s["r"].float()).to(s["r"].dtype)
        r = (h.double().square().mean(-1, keepdim=True) + _EPS).rsqrt().float()
        return [*_plain_quant((h.float() * r) * s["w"].float()), h]
    if k == "linear":
        y = (s["xq"].float() * _wide(s["xs"], s["k"])) @ _weight(s["wq"], s["ws"]).t()
        return (y if s["b"] is None else y + s["b"]).to(_DT[s["out"]])
    if k == "experts":
        return _plain_experts(s)
    if k == "sort":
        offsets, tokens, slots = _sorted(s["ids"], s["experts"])
        if not s["h"]:
            return [offsets, tokens, slots]
        x = s["x"][tokens.clamp_min(0).long()]
        return [offsets, tokens, slots, torch.where(tokens[:, None] < 0, torch.zeros((), dtype=x.dtype, device=x.device), x)]
    return _plain_back(s)


# ------------------------------------------------------------------ 64 bits
def _exact_codes(v):
    """(codes as the values that the format holds, scales) of 64-bit rows."""
    codes, scales = [], []
    for part in v.split(128, -1):
        s = part.abs().amax(-1).clamp_min(1e-12) / 448
        codes.append((part / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).double())
        scales.append(s)
    return torch.cat(codes, -1), torch.stack(scales, -1)


def _exact_product(xq, xs, wq, ws):
    y = xq.new_zeros((xq.shape[0], wq.shape[0]), dtype=torch.float64)
    for b in range(xs.shape[1]):
        cut = slice(128 * b, 128 * b + 128)
        rows = ws[:, b].double()[torch.arange(wq.shape[0], device=wq.device) // 128]
        y += (xq[:, cut].double() @ wq[:, cut].double().t()) * xs[:, b].double()[:, None] * rows
    return y


def exact(case, seed):
    s = prepare(case, seed)
    k = s["kind"]
    if k == "quant":
        if s["op"] == "silu":
            f = s["h"]
            a = s["x"][:, :f].double()
            return _exact_codes(a / (1 + torch.exp(-a)) * s["x"][:, f:].double())
        if s["op"] == "rows":
            return _exact_codes(s["x"].double())
        total = s["x"].double() + s["r"].double()
        h = total.to(s["r"].dtype).double()          # the norm is that of the rows the next layer is given
        return [*_exact_codes(h * s["w"].double() / ((h * h).sum(-1, keepdim=True) / s["h"] + _EPS).sqrt()), total]
    if k == "linear":
        y = _exact_product(s["xq"], s["xs"], s["wq"], s["ws"])
        return y if s["b"] is None else y + s["b"].double()
    ids = s["ids"].tolist()
    if k == "experts":
        rows = [[] for _ in range(s["experts"])]
        for t, row in enumerate(ids):
            for e in row:
                rows[e].append(t)
        out, at = [], 0
        for e, ts in enumerate(rows):
            if ts:
                pick = torch.tensor(ts if s["pick"] else range(at, at + len(ts)), device=DEV)
                out.append(_exact_product(s["xq"].view(torch.uint8)[pick].view(torch.float8_e4m3fn), s["xs"][pick], s["wq"][e], s["ws"][e]))
                at += len(ts)
        return torch.cat(out)
    places = [[] for _ in range(s["experts"])]
    for t, row in enumerate(ids):
        for j, e in enumerate(row):
            if e >= 0:
                places[e].append((t, j))
    order = [p for place in places for p in place]
    if k == "sort":
        offsets, slots = [0], [[-1] * s["top"] for _ in ids]
        for place in places:
            offsets.append(offsets[-1] + len(place))
        for at, (t, j) in enumerate(order):
            slots[t][j] = at
        tokens = [t for t, _ in order] + [-1] * (len(ids) * s["top"] - len(order))
        ints = [torch.tensor(v, dtype=torch.int32, device=DEV) for v in (offsets, tokens, slots)]
        if not s["h"]:
            return ints
        x = torch.zeros((len(tokens), s["h"]), dtype=torch.float64, device=DEV)
        x[:len(order)] = s["x"].double()[torch.tensor(tokens[:len(order)], dtype=torch.long, device=DEV)]
        return [*ints, x]
    at = torch.tensor([t for t, _ in order], device=DEV), torch.tensor([j for _, j in order], device=DEV)
    w, y = s["w"].double()[at], s["y"][:len(order)].double()
    shape = (s["tokens"], s["h"])
    out = [torch.zeros(shape, dtype=torch.float64, device=DEV).index_add_(0, at[0], y * w[:, None])]
    if s["grad"]:
        d = s["dout"].double()[at[0]]
        dy = torch.zeros(s["y"].shape, dtype=torch.float64, device=DEV)
        dy[:len(order)] = d * w[:, None]
        dw = torch.zeros(s["w"].shape, dtype=torch.float64, device=DEV)
        dw[at] = (d * y).sum(-1)
        out += [dy, dw, torch.zeros(shape, dtype=torch.float64, device=DEV).index_add_(0, at[0], dy[:len(order)])]
    return out


def work(case):
    c, k = case, case["kind"]
    if k == "quant":
        v, size = c["m"] * c["h"], _SIZE[c["dt"]]
        ins = {"norm": 3, "silu": 2, "rows": 1}[c["op"]]     # (the norm reads the rows and the residual and writes it)
        return {"bytes": v * (ins * size + 1) + 4 * c["m"] * -(-c["h"] // 128), "flops": 8 * v}
    if k == "linear":
        m, n, d = c["m"], c["n"], c["k"]
        b = -(-d // 128)
        return {"bytes": m * (d + 4 * b) + n * d + 4 * b * -(-n // 128) + (4 * n if c["bias"] else 0) + m * n * _SIZE[c["out"]],
                "flops": 2 * m * n * d}
    t, top, experts = c["tokens"], c["top"], c["experts"]
    pairs = t * top
    if k == "experts":
        n, d = c["n"], c["k"]
        hit = experts * (1 - (1 - top / experts) ** t)       # experts that get a row, were all alike
        b = -(-d // 128)
        return {"bytes": (t if c["pick"] else pairs) * (d + 4 * b) + hit * (n * d + 4 * b * -(-n // 128))
                + pairs * n * _SIZE[c["out"]], "flops": 2 * pairs * n * d}
    row = c["h"] * _SIZE[c["dt"]]
    if k == "sort":
        return {"bytes": 16 * pairs + 4 * experts + (t + pairs) * row, "flops": pairs}
    out = {"bytes": (t + pairs) * row + 8 * pairs, "flops": 2 * pairs * c["h"]}
    if c["grad"]:                                            # the rows and the weights once more, and the rows' own gradient
        out = {"bytes": out["bytes"] + (2 * t + 3 * pairs) * row + 12 * pairs, "flops": 5 * out["flops"] // 2}
    return out
