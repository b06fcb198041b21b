"""Measured calls of the language-model operators (bafe_b200.lm).

Three operators that stand together around a model's matrix products:

* the root-mean-square norm that feeds a product, with the residual's
  addition on the way in and, for 8-bit products, e4m3 output with one scale
  per token; and its gradient;
* products grouped by expert with ragged sizes (16-bit, and e4m3 with the
  norm's scales), with both gradients;
* the product of a few tokens with 4-bit weights that have group scales.

With `own` false, run() computes them from elementary torch operations in
32 bits; with `own` true it makes the calls a user of the framework makes.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_lm = None
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
_E4M3_MAX = 448.0
_EPS = 1e-6


def _framework():
    """The framework's operators, imported on the first call that needs them."""
    global _lm
    if _lm is None:
        root = Path(__file__).resolve().parent.parent
        sys.path.insert(0, str(root / "bafe-basic-algibra-fusion-engine-_b200"))
        from bafe_b200 import lm
        _lm = lm
    return _lm


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # the norm before a product, one generated token: pure latency
        {"name": "norm8 one token", "op": "norm", "rows": 1, "width": 4096, "type": "bf16", "residual": True,
         "to8": True},
        # the same for a long prompt, feeding an 8-bit product
        {"name": "norm8 prompt", "op": "norm", "rows": 8192, "width": 8192, "type": "bf16", "residual": True,
         "to8": True},
        # a width and a row count that divide by nothing, in 32 bits
        {"name": "norm f32 odd", "op": "norm", "rows": 777, "width": 5003, "type": "f32", "residual": False,
         "to8": False},
        # the norm's gradient in training
        {"name": "norm gradient", "op": "norm_grad", "rows": 8192, "width": 4096, "type": "bf16", "residual": True},
        # one token through a square projection held in 4 bits
        {"name": "w4 one token", "op": "w4", "rows": 1, "out": 4096, "in": 4096, "group": 128, "zeros": False,
         "type": "bf16"},
        # eight sequences decoding together through a wide projection, with zero points
        {"name": "w4 eight tokens wide", "op": "w4", "rows": 8, "out": 32768, "in": 8192, "group": 128, "zeros": True,
         "type": "f16"},
        # sizes that end inside a group and inside a tile
        {"name": "w4 odd", "op": "w4", "rows": 3, "out": 1531, "in": 2200, "group": 64, "zeros": True,
         "type": "bf16"},
        # eight tokens spread over eight experts: the weights' bytes are the cost
        {"name": "experts decode", "op": "experts", "rows": 8, "experts": 8, "out": 4096, "in": 4096, "type": "bf16",
         "route": 5},
        # a long prompt over sixteen experts, unevenly loaded
        {"name": "experts prompt", "op": "experts", "rows": 16384, "experts": 16, "out": 4096, "in": 4096,
         "type": "bf16", "route": 2},
        # the same in 8 bits, tokens scaled by row and weights by output channel
        {"name": "experts8 prompt", "op": "experts", "rows": 16384, "experts": 16, "out": 4096, "in": 4096,
         "type": "e4m3", "route": 2},
        # training: the gradient of the tokens ...
        {"name": "experts grad input", "op": "experts_dx", "rows": 8192, "experts": 16, "out": 4096, "in": 2048,
         "type": "bf16", "route": 3},
        # ... and of the weights
        {"name": "experts grad weight", "op": "experts_dw", "rows": 8192, "experts": 16, "out": 4096, "in": 2048,
         "type": "bf16", "route": 3},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "w4", "w4", "experts", "experts", "experts_dx", "experts_dw"])
    if op in ("norm", "norm_grad"):
        c = {"op": op, "rows": _log(rng, 1, 8192), "width": _log(rng, 16, 8192),
             "type": rng.choice(["f32", "bf16", "bf16", "f16"]), "residual": rng.random() < 0.6}
        if op == "norm":
            c["to8"] = rng.random() < 0.5
        if rng.random() < 0.5:
            c["width"] = max(16, c["width"] // 16 * 16)
        return c
    if op == "w4":
        c = {"op": op, "rows": _log(rng, 1, 32), "out": _log(rng, 64, 32768), "in": _log(rng, 64, 8192),
             "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5,
             "type": rng.choice(["bf16", "f16", "e4m3"])}
        if rng.random() < 0.6:
            c["in"] = max(64, c["in"] // 64 * 64)
        return c
    t = rng.choice(["bf16", "bf16", "f16"])
    if op == "experts":
        t = rng.choice(["bf16", "f16", "e4m3"])
    c = {"op": op, "rows": _log(rng, 1, 16384), "experts": _log(rng, 1, 64), "out": _log(rng, 64, 4096),
         "in": _log(rng, 64, 4096), "type": t, "route": rng.randrange(1 << 20)}
    if rng.random() < 0.7:
        c["out"], c["in"] = max(64, c["out"] // 16 * 16), max(64, c["in"] // 16 * 16)
    c["experts"] = max(1, min(c["experts"], (16 * 4096 * 4096) // (c["out"] * c["in"])))
    return c


def _sizes(case):
    """Rows of each expert: uneven as a router's choices are, some of them empty; the same for every seed."""
    rng = random.Random(case["route"])
    share = [rng.expovariate(1.0) * (rng.random() < 0.9) for _ in range(case["experts"])]
    total = sum(share) or 1.0
    if not sum(share):
        share[0] = 1.0
    sizes = [int(case["rows"] * s / total) for s in share]
    for _ in range(case["rows"] - sum(sizes)):
        sizes[rng.randrange(case["experts"])] += 1
    return sizes


# ----------------------------------------------------------------- inputs --

def _to8(v):
    """Rows of v in e4m3 and their scales."""
    scale = v.abs().amax(-1, keepdim=True) / _E4M3_MAX
    return (v / scale).to(torch.float8_e4m3fn), scale.squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    op, t = case["op"], _DT[case["type"]]
    s = {"case": case}
    if op in ("norm", "norm_grad"):
        rows, width = case["rows"], case["width"]
        gain = 0.3 + 0.7 * torch.rand(width, generator=g, device="cuda")     # channels differ in size
        s["weight"] = (1.0 + 0.1 * randn(width)).to(t)
        if op == "norm":
            s["x"] = (randn(rows, width) * gain).to(t)
            s["residual"] = (3.0 * randn(rows, width) * gain).to(t) if case["residual"] else None
        else:
            s["h"] = (3.0 * randn(rows, width) * gain).to(t)
            s["dy"] = (0.1 * randn(rows, width)).to(t)
            s["dh"] = (0.1 * randn(rows, width)).to(t) if case["residual"] else None
    elif op == "w4":
        rows, n, k, group = case["rows"], case["out"], case["in"], case["group"]
        groups = -(-k // group)
        x = randn(rows, k)
        if case["type"] == "e4m3":
            s["x"], s["x_scale"] = _to8(x)
        else:
            s["x"], s["x_scale"] = x.to(t), None
        half = torch.float16 if case["type"] == "f16" else torch.bfloat16
        q = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
        s["qweight"] = q
        s["scales"] = (0.004 + 0.012 * torch.rand(n, groups, generator=g, device="cuda")).to(half)
        s["zeros"] = (torch.randint(5, 11, (n, groups), generator=g, device="cuda", dtype=torch.uint8)
                      if case["zeros"] else None)
    else:
        rows, e, n, k = case["rows"], case["experts"], case["out"], case["in"]
        sizes = _sizes(case)
        ends = [0]
        for z in sizes:
            ends.append(ends[-1] + z)
        s["sizes"] = sizes
        s["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        w = None
        if op != "experts_dw":
            w = torch.empty(e, n, k, device="cuda", dtype=t if case["type"] != "e4m3" else torch.float8_e4m3fn)
            ws = torch.empty(e, n, device="cuda")
            for i in range(e):
                v = randn(n, k) / math.sqrt(k)
                if case["type"] == "e4m3":
                    w[i], ws[i] = _to8(v)
                else:
                    w[i] = v.to(t)
            s["w"] = w
            s["w_scale"] = ws if case["type"] == "e4m3" else None
        if op in ("experts", "experts_dw"):
            x = randn(rows, k)
            if case["type"] == "e4m3":
                s["x"], s["x_scale"] = _to8(x)
            else:
                s["x"], s["x_scale"] = x.to(t), None
        if op in ("experts_dx", "experts_dw"):
            s["dy"] = (0.1 * randn(rows, n)).to(t)
    return s


# ------------------------------------------------------------------- runs --

def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        lm = _framework()
        if op == "norm":
            if case["to8"]:
                return lm.rms_norm_e4m3(s["x"], s["weight"], s["residual"], eps=_EPS)
            return lm.rms_norm(s["x"], s["weight"], s["residual"], eps=_EPS)
        if op == "norm_grad":
            return lm.rms_norm_grad(s["dy"], s["h"], s["weight"], s["dh"], eps=_EPS)
        if op == "w4":
            return lm.matvec_w4(s["x"], s["qweight"], s["scales"], s["zeros"], group=case["group"],
                                x_scale=s["x_scale"])
        if op == "experts":
            return lm.grouped_matmul(s["x"], s["w"], s["offsets"], x_scale=s["x_scale"], w_scale=s["w_scale"])
        if op == "experts_dx":
            return lm.grouped_matmul_grad_input(s["dy"], s["w"], s["offsets"])
        return lm.grouped_matmul_grad_weight(s["dy"], s["x"], s["offsets"])
    return _PLAIN[op](s, case)


def _plain_norm(s, case):
    x, res, w = s["x"], s["residual"], s["weight"].float()
    if res is not None:
        h16 = (x.float() + res.float()).to(x.dtype)          # the stored sum is what is normalised
    else:
        h16 = x
    h = h16.float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS) * w
    out = []
    if case["to8"]:
        scale = y.abs().amax(-1, keepdim=True) / _E4M3_MAX
        scale = torch.where(scale > 0, scale, torch.ones_like(scale))
        out += [(y / scale).to(torch.float8_e4m3fn), scale.squeeze(-1)]
    else:
        out += [y.to(x.dtype)]
    if res is not None:
        out += [h16]
    return out[0] if len(out) == 1 else tuple(out)


def _plain_norm_grad(s, case):
    dy, h, w = s["dy"].float(), s["h"].float(), s["weight"].float()
    r = torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS)
    g = dy * w
    dx = r * g - h * (r * r * r) * (g * h).mean(-1, keepdim=True)
    if s["dh"] is not None:
        dx = dx + s["dh"].float()
    dw = (dy * h * r).sum(0)
    return dx.to(s["h"].dtype), dw.to(s["weight"].dtype)


def _w4_weight(s, case, t):
    """The 4-bit weights as numbers of type t: (q - zero) * scale."""
    n, k, group = case["out"], case["in"], case["group"]
    q = torch.stack((s["qweight"] & 15, s["qweight"] >> 4), -1).reshape(n, -1)[:, :k].to(t)
    z = s["zeros"].to(t) if s["zeros"] is not None else torch.full_like(s["scales"], 8.0, dtype=t)
    z = z.repeat_interleave(group, 1)[:, :k]
    return (q - z) * s["scales"].to(t).repeat_interleave(group, 1)[:, :k]


def _plain_w4(s, case):
    y = s["x"].float() @ _w4_weight(s, case, torch.float32).t()
    if s["x_scale"] is not None:
        y = y * s["x_scale"][:, None]
    return y.to(s["scales"].dtype)


def _blocks(s):
    """(expert, first row, end) of the experts that have rows; the loop over them is the plain form's grouping."""
    at = 0
    for e, z in enumerate(s["sizes"]):
        if z:
            yield e, at, at + z
        at += z


def _plain_experts(s, case):
    e8 = case["type"] == "e4m3"
    y = torch.empty(case["rows"], case["out"], device=s["x"].device,
                    dtype=torch.bfloat16 if e8 else s["x"].dtype)
    for e, a, b in _blocks(s):
        v = s["x"][a:b].float() @ s["w"][e].float().t()
        if e8:
            v = v * s["x_scale"][a:b, None] * s["w_scale"][e]
        y[a:b] = v.to(y.dtype)
    return y


def _plain_experts_dx(s, case):
    dx = torch.empty(case["rows"], case["in"], device=s["dy"].device, dtype=s["dy"].dtype)
    for e, a, b in _blocks(s):
        dx[a:b] = (s["dy"][a:b].float() @ s["w"][e].float()).to(dx.dtype)
    return dx


def _plain_experts_dw(s, case):
    dw = torch.zeros(case["experts"], case["out"], case["in"], device=s["dy"].device, dtype=s["dy"].dtype)
    for e, a, b in _blocks(s):
        dw[e] = (s["dy"][a:b].float().t() @ s["x"][a:b].float()).to(dw.dtype)
    return dw


_PLAIN = {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "w4": _plain_w4, "experts": _plain_experts,
          "experts_dx": _plain_experts_dx, "experts_dw": _plain_experts_dw}


# ------------------------------------------------------------------- work --

def work(case):
    op, b = case["op"], _BYTES[case["type"]]
    if op == "norm":
        n = case["rows"] * case["width"]
        out = n * (1 if case["to8"] else b) + (4 * case["rows"] if case["to8"] else 0)
        return {"bytes": n * b * (3 if case["residual"] else 1) + out + case["width"] * b, "flops": 4 * n}
    if op == "norm_grad":
        n = case["rows"] * case["width"]
        return {"bytes": n * b * (4 if case["residual"] else 3) + 2 * case["width"] * b, "flops": 10 * n}
    if op == "w4":
        m, n, k = case["rows"], case["out"], case["in"]
        groups = -(-k // case["group"])
        by = n * ((k + 1) // 2) + n * groups * (3 if case["zeros"] else 2) + m * k * b + m * n * 2
        return {"bytes": by + (4 * m if case["type"] == "e4m3" else 0), "flops": 2 * m * n * k}
    m, n, k = case["rows"], case["out"], case["in"]
    active = sum(1 for z in _sizes(case) if z)
    offsets = 4 * (case["experts"] + 1)
    if op == "experts":
        by = m * k * b + active * n * k * b + m * n * 2
        if case["type"] == "e4m3":
            by += 4 * m + 4 * active * n
    elif op == "experts_dx":
        by = m * n * b + active * n * k * b + m * k * b
    else:
        by = m * n * b + m * k * b + case["experts"] * n * k * b
    return {"bytes": by + offsets, "flops": 2 * m * n * k}


# ------------------------------------------------------------------ exact --

def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    d = torch.float64
    if op == "norm":
        h = s["x"].to(d)
        if s["residual"] is not None:
            h = (h + s["residual"].to(d)).to(s["x"].dtype).to(d)      # rounded as it is stored: part of the definition
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["width"] + _EPS) * s["weight"].to(d)
        if case["to8"]:
            top = y.abs().max(-1, keepdim=True).values
            scale = torch.where(top > 0, top / _E4M3_MAX, torch.ones_like(top))
            out = [y / scale, scale[:, 0]]
        else:
            out = [y]
        if s["residual"] is not None:
            out.append(h)
        return out[0] if len(out) == 1 else tuple(out)
    if op == "norm_grad":
        dy, h, w = s["dy"].to(d), s["h"].to(d), s["weight"].to(d)
        rms = torch.sqrt((h * h).sum(-1, keepdim=True) / case["width"] + _EPS)
        n = h / rms
        g = dy * w
        dx = (g - n * (g * n).sum(-1, keepdim=True) / case["width"]) / rms
        if s["dh"] is not None:
            dx = dx + s["dh"].to(d)
        return dx, (dy * n).sum(0)
    if op == "w4":
        n, k, group = case["out"], case["in"], case["group"]
        at = torch.arange(k, device="cuda")
        rows = []
        for a in range(0, n, 4096):                               # a slab of outputs at a time bounds the memory
            byte = s["qweight"][a:a + 4096][:, at // 2].to(torch.int32)
            q = ((byte >> (4 * (at % 2)).to(torch.int32)) & 15).to(d)
            z = s["zeros"][a:a + 4096][:, at // group].to(d) if s["zeros"] is not None else 8.0
            rows.append(s["x"].to(d) @ ((q - z) * s["scales"][a:a + 4096][:, at // group].to(d)).t())
        y = torch.cat(rows, 1)
        return y * s["x_scale"].to(d)[:, None] if s["x_scale"] is not None else y
    at = 0
    if op == "experts":
        parts = []
        for e, z in enumerate(s["sizes"]):
            x = s["x"][at:at + z].to(d)
            w = s["w"][e].to(d)
            if case["type"] == "e4m3":
                x, w = x * s["x_scale"][at:at + z, None].to(d), w * s["w_scale"][e][:, None].to(d)
            parts.append(torch.mm(x, w.t()))
            at += z
        return torch.cat(parts)
    if op == "experts_dx":
        parts = []
        for e, z in enumerate(s["sizes"]):
            parts.append(torch.mm(s["dy"][at:at + z].to(d), s["w"][e].to(d)))
            at += z
        return torch.cat(parts)
    parts = []
    for z in s["sizes"]:
        parts.append(torch.mm(s["dy"][at:at + z].to(d).t(), s["x"][at:at + z].to(d)))
        at += z
    return torch.stack(parts)
