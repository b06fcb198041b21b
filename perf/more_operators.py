"""Measured calls of the routing and loss operators (bafe_b200.lm).

Two sets that stand at the two ends of the grouped products:

* the router that chooses each token's experts and lays out the rows by
  expert, with its gradient; the rows' way to the experts and back (gather,
  weighted sum), with its gradient;
* softmax cross entropy over a large vocabulary straight from the hidden
  states and the output weights, in pieces of the vocabulary and without
  keeping the logits, and its gradient.

With `own` false, run() computes them from elementary torch operations in 32
bits, the order of the routers' scores in 64; with `own` true it makes the
calls a user of the framework makes.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_lm = None
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_IGNORE = -100


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
        # one generated token before many small experts, in groups, with a balance bias: pure latency
        {"name": "route one token", "op": "route", "rows": 1, "experts": 256, "k": 8, "score": "sigmoid", "groups": 8,
         "keep": 4, "bias": True, "renorm": True, "type": "f32", "padded": 0.0},
        # the same router over a long prompt
        {"name": "route prompt", "op": "route", "rows": 16384, "experts": 256, "k": 8, "score": "sigmoid", "groups": 8,
         "keep": 4, "bias": True, "renorm": True, "type": "f32", "padded": 0.0},
        # softmax scores over a count of experts that is no power of two, 16-bit logits, a padded batch
        {"name": "route odd padded", "op": "route", "rows": 4001, "experts": 60, "k": 4, "score": "softmax", "groups": 1,
         "keep": 1, "bias": False, "renorm": False, "type": "bf16", "padded": 0.2},
        # the router's gradient in training
        {"name": "route gradient", "op": "route_grad", "rows": 8192, "experts": 64, "k": 6, "score": "softmax",
         "renorm": False, "type": "f32"},
        # a prompt's rows, laid out by expert
        {"name": "dispatch prompt", "op": "dispatch", "rows": 8192, "width": 4096, "experts": 64, "k": 8, "type": "bf16"},
        # one token's experts summed: latency
        {"name": "combine one token", "op": "combine", "rows": 1, "width": 4096, "experts": 64, "k": 8, "type": "bf16",
         "weighted": True},
        # a prompt's
        {"name": "combine prompt", "op": "combine", "rows": 8192, "width": 4096, "experts": 64, "k": 8, "type": "bf16",
         "weighted": True},
        # its gradient in training, with the weights'
        {"name": "combine gradient", "op": "combine_grad", "rows": 4096, "width": 2048, "experts": 64, "k": 6,
         "type": "bf16"},
        # the loss of a few tokens: the weights' bytes are the cost
        {"name": "loss few rows", "op": "loss", "rows": 16, "width": 4096, "vocab": 32768, "type": "bf16"},
        # a training batch over a large vocabulary
        {"name": "loss batch", "op": "loss", "rows": 8192, "width": 4096, "vocab": 131072, "type": "bf16"},
        # the gradient of a training batch
        {"name": "loss gradient", "op": "loss_grad", "rows": 8192, "width": 4096, "vocab": 32768, "type": "bf16"},
        # sizes that end inside every tile, rows of the weights off 16-byte boundaries
        {"name": "loss gradient odd", "op": "loss_grad", "rows": 777, "width": 1150, "vocab": 50001, "type": "f16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "route", "route", "route_grad", "dispatch", "combine", "combine", "combine_grad", "loss",
                     "loss", "loss_grad", "loss_grad"])
    if op in ("route", "route_grad"):
        experts = _log(rng, 4, 512)
        c = {"op": op, "rows": _log(rng, 1, 16384), "k": min(experts, rng.randint(1, 10)),
             "score": rng.choice(["softmax", "sigmoid"]), "renorm": rng.random() < 0.6,
             "type": rng.choice(["f32", "f32", "bf16", "f16"])}
        if op == "route":
            c.update(groups=1, keep=1, bias=rng.random() < 0.5, padded=rng.choice([0.0, 0.0, rng.random()]))
            if rng.random() < 0.5 and experts >= 16:
                c["groups"] = rng.choice([2, 4, 5, 8])
                experts = experts // c["groups"] * c["groups"]
                c["keep"] = rng.randint(1, c["groups"])
                c["k"] = min(c["k"], experts // c["groups"] * c["keep"])
        c["experts"] = experts
        return c
    if op in ("dispatch", "combine", "combine_grad"):
        c = {"op": op, "rows": _log(rng, 1, 8192), "width": _log(rng, 32, 4096), "experts": _log(rng, 8, 256),
             "k": rng.randint(1, 8), "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
        if rng.random() < 0.6:
            c["width"] = max(32, c["width"] // 32 * 32)
        if op == "combine":
            c["weighted"] = rng.random() < 0.7
        return c
    c = {"op": op, "rows": _log(rng, 1, 8192), "width": _log(rng, 64, 4096), "vocab": _log(rng, 256, 131072),
         "type": rng.choice(["bf16", "bf16", "f16"])}
    if rng.random() < 0.7:
        c["width"] = max(64, c["width"] // 64 * 64)
    return c


# ----------------------------------------------------------------- inputs --

def _chosen(rows, experts, k, g):
    """k different experts for each row, some experts more often than others."""
    lean = 0.5 * torch.randn(experts, generator=g, device="cuda")
    u = torch.rand(rows, experts, generator=g, device="cuda").clamp_min(1e-9)
    return torch.topk(lean - torch.log(-torch.log(u)), k, -1).indices


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    op, rows, t = case["op"], case["rows"], _DT[case["type"]]
    s = {"case": case}
    if op in ("route", "route_grad"):
        e, k = case["experts"], case["k"]
        logits = randn(rows, e) + 0.5 * randn(e)
        if op == "route":
            if case["padded"]:
                logits[torch.rand(rows, generator=g, device="cuda") < case["padded"]] = -math.inf
            s["bias"] = 0.1 * randn(e) if case["bias"] else None
            s["logits"] = logits.to(t)
        else:
            s["logits"] = logits.to(t)
            s["experts"] = torch.sort(s["logits"], dim=-1, descending=True, stable=True).indices[:, :k].int().contiguous()
            s["dweights"] = 0.1 * randn(rows, k)
        return s
    if op in ("dispatch", "combine", "combine_grad"):
        width, k = case["width"], min(case["k"], case["experts"])
        flat = _chosen(rows, case["experts"], k, g).reshape(-1)
        source = torch.sort(flat, stable=True).indices
        place = torch.empty_like(source)
        place[source] = torch.arange(rows * k, device="cuda")
        s["place"] = place.int().view(rows, k)
        if op == "dispatch":
            s["x"] = randn(rows, width).to(t)
            return s
        s["y"] = randn(rows * k, width).to(t)
        s["weights"] = None
        if op == "combine_grad" or case["weighted"]:
            s["weights"] = torch.softmax(randn(rows, k), -1)
        if op == "combine_grad":
            s["dout"] = (0.1 * randn(rows, width)).to(t)
        return s
    d, v = case["width"], case["vocab"]
    s["x"] = randn(rows, d).to(t)
    w = torch.empty(v, d, device="cuda", dtype=t)
    for a in range(0, v, 16384):
        w[a:a + 16384] = (randn(min(16384, v - a), d) * (2.0 / math.sqrt(d))).to(t)
    s["w"] = w
    target = torch.randint(0, v, (rows,), generator=g, device="cuda")
    s["target"] = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.05, _IGNORE, target)   # padding, prompts
    if op == "loss_grad":
        _, s["lse"] = _plain_loss(s, case)
        s["dloss"] = torch.full((rows,), 1.0 / max(1, rows), device="cuda")       # of the mean over the batch
    return s


# ------------------------------------------------------------------- runs --

def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        lm = _framework()
        if op == "route":
            return tuple(lm.route(s["logits"], case["k"], score=case["score"], bias=s["bias"], groups=case["groups"],
                                  keep_groups=case["keep"], renormalize=case["renorm"]))
        if op == "route_grad":
            return lm.route_grad(s["dweights"], s["logits"], s["experts"], score=case["score"],
                                 renormalize=case["renorm"])
        if op == "dispatch":
            return lm.dispatch(s["x"], s["place"])
        if op == "combine":
            return lm.combine(s["y"], s["place"], s["weights"])
        if op == "combine_grad":
            return lm.combine_grad(s["dout"], s["y"], s["place"], s["weights"])
        if op == "loss":
            return lm.linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=_IGNORE)
        return lm.linear_cross_entropy_grad(s["dloss"], s["x"], s["w"], s["target"], s["lse"], ignore_index=_IGNORE)
    return _PLAIN[op](s, case)


def _plain_scores(logits, score):
    """The scores in 64 bits: the choice hangs on their order."""
    z = logits.double()
    open_ = z > -math.inf
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z)), open_
    top = z.max(-1, keepdim=True).values
    e = torch.exp(z - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total)), open_


def _plain_route(s, case):
    logits, k, e = s["logits"], case["k"], case["experts"]
    rows, groups = case["rows"], case["groups"]
    scores, open_ = _plain_scores(logits, case["score"])
    key = scores if s["bias"] is None else scores + s["bias"].double()
    key = torch.where(open_, key, torch.full_like(key, -math.inf))
    if groups > 1:
        best = torch.sort(key.view(rows, groups, e // groups), dim=-1, descending=True).values[..., :2]
        total = torch.where(best > -math.inf, best, torch.zeros_like(best)).sum(-1)
        total = torch.where(best[..., 0] > -math.inf, total, torch.full_like(total, -math.inf))
        order = torch.sort(total, dim=-1, descending=True, stable=True).indices[:, :case["keep"]]
        keep = torch.zeros(rows, groups, dtype=torch.bool, device=key.device).scatter_(1, order, True)
        key = torch.where(keep.repeat_interleave(e // groups, 1), key, torch.full_like(key, -math.inf))
    top, at = torch.sort(key, dim=-1, descending=True, stable=True)
    top, at = top[:, :k], at[:, :k]
    some = top > -math.inf
    w = torch.where(some, scores.gather(1, at), torch.zeros_like(top))
    if case["renorm"]:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
    experts = torch.where(some, at, torch.full_like(at, -1)).int()
    # the rows' order by expert
    flat = experts.reshape(-1)
    label = torch.where(flat < 0, torch.full_like(flat, e), flat)
    label, source = torch.sort(label, stable=True)
    offsets = torch.searchsorted(label, torch.arange(e + 1, device=flat.device, dtype=flat.dtype)).int()
    place = torch.empty_like(flat)
    inside = label < e
    place[source] = torch.where(inside, torch.arange(rows * k, device=flat.device), -1).int()
    return w.float(), experts, offsets, place.view(rows, k)


def _plain_route_grad(s, case):
    z, at, g = s["logits"].float(), s["experts"].long(), s["dweights"]
    if case["score"] == "softmax":
        p = torch.exp(z - z.max(-1, keepdim=True).values)
        p = p / p.sum(-1, keepdim=True)
        slope = 1.0
    else:
        p = 1.0 / (1.0 + torch.exp(-z))
        slope = 1.0 - p
    ds = torch.zeros_like(z)
    if case["renorm"]:
        chosen = p.gather(1, at)
        total = chosen.sum(-1, keepdim=True)
        w = chosen / total
        ds.scatter_(1, at, (g - (g * w).sum(-1, keepdim=True)) / total)
    else:
        ds.scatter_(1, at, g)
    if case["score"] == "softmax":
        dz = p * (ds - (p * ds).sum(-1, keepdim=True))
    else:
        dz = ds * p * slope
    return dz.to(s["logits"].dtype)


def _plain_dispatch(s, case):
    place = s["place"].long()
    y = s["x"].new_empty(place.numel(), case["width"])
    y[place.reshape(-1)] = s["x"].repeat_interleave(place.shape[1], 0)
    return y


def _plain_combine(s, case):
    place = s["place"].long()
    out = None
    for j in range(place.shape[1]):
        v = s["y"][place[:, j]].float()
        if s["weights"] is not None:
            v = v * s["weights"][:, j:j + 1]
        out = v if out is None else out + v
    return out.to(s["y"].dtype)


def _plain_combine_grad(s, case):
    place, dout = s["place"].long(), s["dout"].float()
    dy = torch.empty_like(s["y"])
    dw = torch.empty_like(s["weights"])
    for j in range(place.shape[1]):
        dw[:, j] = (dout * s["y"][place[:, j]].float()).sum(-1)
        dy[place[:, j]] = (dout * s["weights"][:, j:j + 1]).to(dy.dtype)
    return dy, dw


_PIECE = 16384


def _plain_loss(s, case):
    x, w, target = s["x"].float(), s["w"], s["target"]
    rows = x.shape[0]
    top = torch.full((rows,), -math.inf, device=x.device)
    total = torch.zeros(rows, device=x.device)
    hit = torch.zeros(rows, device=x.device)
    for a in range(0, w.shape[0], _PIECE):
        z = x @ w[a:a + _PIECE].float().t()
        m = torch.maximum(top, z.max(-1).values)
        total = total * torch.exp(top - m) + torch.exp(z - m[:, None]).sum(-1)
        top = m
        here = (target >= a) & (target < a + z.shape[1])
        at = torch.where(here, target - a, torch.zeros_like(target))
        hit = torch.where(here, z.gather(1, at[:, None])[:, 0], hit)
    lse = top + torch.log(total)
    return torch.where(target == _IGNORE, torch.zeros_like(lse), lse - hit), lse


def _plain_loss_grad(s, case):
    x, w, target, lse = s["x"].float(), s["w"], s["target"], s["lse"]
    scale = torch.where(target == _IGNORE, torch.zeros_like(lse), s["dloss"])
    dx = torch.zeros_like(x)
    dw = torch.empty_like(w)
    for a in range(0, w.shape[0], _PIECE):
        part = w[a:a + _PIECE].float()
        g = torch.exp(x @ part.t() - lse[:, None])
        here = (target >= a) & (target < a + part.shape[0])
        at = torch.where(here, target - a, torch.zeros_like(target))
        g.scatter_add_(1, at[:, None], torch.where(here, -1.0, 0.0)[:, None])
        g *= scale[:, None]
        dx += g @ part
        dw[a:a + _PIECE] = (g.t() @ x).to(dw.dtype)
    return dx.to(s["x"].dtype), dw


_PLAIN = {"route": _plain_route, "route_grad": _plain_route_grad, "dispatch": _plain_dispatch, "combine": _plain_combine,
          "combine_grad": _plain_combine_grad, "loss": _plain_loss, "loss_grad": _plain_loss_grad}


# ------------------------------------------------------------------- work --

def work(case):
    op, b, rows = case["op"], _BYTES[case["type"]], case["rows"]
    if op == "route":
        e, k = case["experts"], case["k"]
        return {"bytes": rows * e * b + (4 * e if case["bias"] else 0) + 12 * rows * k + 4 * (e + 1),
                "flops": 8 * rows * e}
    if op == "route_grad":
        e, k = case["experts"], case["k"]
        read = k if case["renorm"] or case["score"] == "sigmoid" else e      # only the chosen ones matter
        return {"bytes": rows * b * (read + e) + 8 * rows * k, "flops": 8 * rows * e}
    if op in ("dispatch", "combine", "combine_grad"):
        k, w = min(case["k"], case["experts"]), case["width"]
        if op == "combine_grad":
            return {"bytes": rows * w * b * (1 + 2 * k) + 12 * rows * k, "flops": 3 * rows * k * w}
        weights = 4 * rows * k if op == "combine" and case["weighted"] else 0
        return {"bytes": rows * w * b * (1 + k) + 4 * rows * k + weights, "flops": 2 * rows * k * w if op == "combine" else 0}
    d, v = case["width"], case["vocab"]
    if op == "loss":
        return {"bytes": (rows + v) * d * b + 16 * rows, "flops": 2 * rows * v * d}
    return {"bytes": 2 * (rows + v) * d * b + 16 * rows, "flops": 6 * rows * v * d}


# ------------------------------------------------------------------ exact --

def _exact_route(s, case):
    """The choice one expert after the other; the places by counting."""
    z = s["logits"].to(torch.float64)
    rows, e = z.shape
    k, groups, dev = case["k"], case["groups"], z.device
    shut = torch.isneginf(z)
    if case["score"] == "softmax":
        norm = torch.logsumexp(z, -1, keepdim=True)
        p = torch.where(shut, 0.0, torch.exp(z - torch.where(torch.isneginf(norm), 0.0, norm)))
    else:
        p = torch.where(shut, 0.0, torch.special.expit(z))
    key = torch.where(shut, -math.inf, p + (s["bias"].to(torch.float64) if s["bias"] is not None else 0.0))
    number = torch.arange(e, device=dev)
    line = torch.arange(rows, device=dev)

    def first_best(values):
        """Index of each row's largest value, the lowest of equals."""
        n = values.shape[1]
        best = values == values.amax(-1, keepdim=True)
        return torch.where(best, torch.arange(n, device=dev), n).amin(-1)

    if groups > 1:
        size = e // groups
        worth = torch.empty(rows, groups, dtype=torch.float64, device=dev)
        for j in range(groups):
            part = key[:, j * size:(j + 1) * size].clone()
            one = part.amax(-1)
            part[line, first_best(part)] = -math.inf
            two = part.amax(-1) if size > 1 else torch.full_like(one, -math.inf)
            worth[:, j] = torch.where(torch.isneginf(two), one, one + two)
        kept = torch.zeros(rows, groups, dtype=torch.bool, device=dev)
        for _ in range(case["keep"]):
            # groups without an open expert are worth -inf; which of them is taken changes nothing
            j = first_best(worth)
            kept[line, j] = True
            worth[line, j] = -math.inf
        key = torch.where(kept[:, number // size], key, -math.inf)
    experts = torch.full((rows, k), -1, dtype=torch.int64, device=dev)
    weights = torch.zeros(rows, k, dtype=torch.float64, device=dev)
    for j in range(k):
        at = first_best(key)
        some = ~torch.isneginf(key[line, at])
        experts[:, j] = torch.where(some, at, -1)
        weights[:, j] = torch.where(some, p[line, at], 0.0)
        key[line, at] = -math.inf
    if case["renorm"]:
        weights = weights / weights.sum(-1, keepdim=True).clamp_min(1e-300)
    flat = experts.reshape(-1)
    offsets = torch.zeros(e + 1, dtype=torch.int64, device=dev)
    place = torch.full_like(flat, -1)
    at = 0
    for j in range(e):
        mine = torch.nonzero(flat == j)[:, 0]
        offsets[j] = at
        place[mine] = torch.arange(at, at + len(mine), device=dev)
        at += len(mine)
    offsets[e] = at
    return weights, experts, offsets, place.view(rows, k)


def _exact_route_grad(s, case):
    z = s["logits"].to(torch.float64).requires_grad_()
    p = torch.softmax(z, -1) if case["score"] == "softmax" else torch.sigmoid(z)
    w = torch.gather(p, 1, s["experts"].to(torch.int64))
    if case["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return torch.autograd.grad((w * s["dweights"].to(torch.float64)).sum(), z)[0]


def _exact_loss(s, case):
    x, w, target = s["x"].to(torch.float64), s["w"], s["target"]
    parts, hit = [], torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    for a in range(0, w.shape[0], 8192):
        parts.append(torch.logsumexp(torch.mm(x, w[a:a + 8192].to(torch.float64).t()), -1))
    for a in range(0, x.shape[0], 1024):
        rows = w[target[a:a + 1024].clamp_min(0)].to(torch.float64)
        hit[a:a + 1024] = torch.einsum("rd,rd->r", x[a:a + 1024], rows)
    lse = torch.logsumexp(torch.stack(parts), 0)
    return (lse - hit) * (target != _IGNORE), lse


def _exact_loss_grad(s, case):
    x, w, target = s["x"].to(torch.float64), s["w"], s["target"]
    dloss = s["dloss"].to(torch.float64) * (target != _IGNORE)
    dx = torch.zeros_like(x)
    dw = []
    for a in range(0, w.shape[0], 8192):
        part = w[a:a + 8192].to(torch.float64)
        column = torch.arange(a, a + part.shape[0], device=x.device)
        g = torch.exp(torch.mm(x, part.t()) - s["lse"].to(torch.float64)[:, None])
        g = (g - (target[:, None] == column).to(torch.float64)) * dloss[:, None]
        dx.addmm_(g, part)
        dw.append(torch.mm(g.t(), x))
    return dx, torch.cat(dw)


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    d = torch.float64
    if op == "route":
        return _exact_route(s, case)
    if op == "route_grad":
        return _exact_route_grad(s, case)
    if op == "loss":
        return _exact_loss(s, case)
    if op == "loss_grad":
        return _exact_loss_grad(s, case)
    if op == "dispatch":
        number = torch.argsort(s["place"].reshape(-1))            # the inverse of place
        token = torch.div(number, s["place"].shape[1], rounding_mode="floor")
        return torch.index_select(s["x"], 0, token).to(d)
    place = s["place"].to(torch.int64)
    rows, k = place.shape
    y = torch.index_select(s["y"], 0, place.reshape(-1)).view(rows, k, -1)
    weights = torch.ones(rows, k, dtype=d, device="cuda") if s["weights"] is None else s["weights"].to(d)
    step = max(1, (1 << 28) // (k * case["width"]))               # bounds the memory
    if op == "combine":
        return torch.cat([torch.einsum("rkw,rk->rw", y[a:a + step].to(d), weights[a:a + step])
                          for a in range(0, rows, step)])
    dout = s["dout"].to(d)
    dy = torch.empty(rows * k, case["width"], dtype=d, device="cuda")
    dy[place.reshape(-1)] = (weights[..., None] * dout[:, None]).view(rows * k, -1)
    return dy, torch.cat([torch.einsum("rkw,rw->rk", y[a:a + step].to(d), dout[a:a + step])
                          for a in range(0, rows, step)])
