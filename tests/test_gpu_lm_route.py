"""Routing to experts (lm.route, lm.route_grad) against the definition in 64
bits: the choices, their order and the places bit for bit, weights and
gradients within derived bounds.

Bounds.  A weight is made of exponentials (an ulp each, and the rounding of
their argument: up to |l - m| half ulps), a sum of up to 1024 of them (32 in a
lane, 5 levels of lanes) and a division; with logits differing by at most 40
that is below 128 ulps, 2^-17 of the weight.  A gradient is p (g - dot): twice
that of p (|g| + sum p |g|), and the rounding to the logits' type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF = math.inf
REL = 2.0 ** -17


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def reference(logits, k, score="softmax", bias=None, groups=1, keep_groups=1, group_top=2, renormalize=True, scale=1.0):
    """Row by row on the CPU, in 64 bits."""
    z = logits.double().cpu()
    b = torch.zeros(z.shape[1], dtype=torch.float64) if bias is None else bias.double().cpu()
    rows, n = z.shape
    weights = torch.zeros(rows, k, dtype=torch.float64)
    experts = torch.full((rows, k), -1, dtype=torch.int32)
    for t in range(rows):
        m = float(z[t].max())
        if score == "softmax":
            e = [math.exp(float(v) - m) if v > -INF else 0.0 for v in z[t]]
            total = math.fsum(e)
            s = [v / total if total else 0.0 for v in e]
        else:
            s = [1.0 / (1.0 + math.exp(-float(v))) if v > -700 else 0.0 for v in z[t]]
        open_ = {i for i in range(n) if z[t, i] > -INF and b[i] > -INF}
        c = [s[i] + float(b[i]) for i in range(n)]
        if bias is None and groups == 1:
            c = [float(v) for v in z[t]]                 # the same order, also where scores underflow
        size = n // groups
        if groups > 1:
            worth = []
            for h in range(groups):
                best = sorted((c[i] for i in range(h * size, (h + 1) * size) if i in open_), reverse=True)[:group_top]
                worth.append(sum(best) if best else -INF)
            kept = sorted(range(groups), key=lambda h: (-worth[h], h))[:keep_groups]
            open_ = {i for i in open_ if i // size in kept}
        order = sorted(open_, key=lambda i: (-c[i], i))[:k]
        total = math.fsum(s[i] for i in order) if renormalize else 1.0
        for j, i in enumerate(order):
            experts[t, j] = i
            weights[t, j] = s[i] / total * scale
    flat = experts.reshape(-1).tolist()
    offsets, place = [0], [-1] * len(flat)
    for e in range(n):
        at = offsets[-1]
        for q, v in enumerate(flat):
            if v == e:
                place[q] = at
                at += 1
        offsets.append(at)
    return weights, experts, torch.tensor(offsets, dtype=torch.int32), torch.tensor(place, dtype=torch.int32).view(rows, k)


def compare(got, want):
    torch.cuda.synchronize()
    assert torch.equal(got.experts.cpu(), want[1])
    assert torch.equal(got.offsets.cpu(), want[2])
    assert torch.equal(got.place.cpu(), want[3])
    err = (got.weights.cpu().double() - want[0]).abs()
    assert (err <= REL * want[0].abs()).all(), float((err / want[0].abs().clamp_min(1e-300)).max())


@pytest.mark.parametrize("rows,n,k,kw", [
    (1, 1, 1, {}),
    (3, 5, 5, dict(renormalize=False)),
    (64, 60, 4, dict(score="softmax", renormalize=False, scale=2.5)),
    (65, 60, 4, dict(score="sigmoid")),
    (7, 256, 8, dict(score="sigmoid", bias=True, groups=8, keep_groups=4)),
    (200, 256, 8, dict(score="sigmoid", bias=True, groups=8, keep_groups=4, renormalize=False)),
    (130, 160, 6, dict(score="softmax", groups=8, keep_groups=3, group_top=1)),
    (130, 160, 6, dict(score="softmax", bias=True, groups=5, keep_groups=2)),
    (33, 96, 3, dict(score="sigmoid", groups=32, keep_groups=1)),
    (33, 24, 3, dict(score="softmax", groups=24, keep_groups=3, bias=True)),
    (40, 63, 7, dict(score="softmax", groups=3, keep_groups=3, bias=True)),
    (100, 512, 22, dict(score="sigmoid", bias=True)),
    (70, 1024, 31, dict(score="softmax", bias=True, groups=4, keep_groups=2)),
    (3, 1024, 31, dict(score="sigmoid", bias=True, groups=32, keep_groups=32)),
    (2, 33, 31, dict(score="softmax")),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_route(cuda, rows, n, k, kw, dtype):
    from bafe_b200 import lm
    g = gen(rows * 1000 + n)
    logits = (2.0 * torch.randn(rows, n, generator=g, device="cuda")).to(dtype)
    kw = dict(kw)
    if kw.pop("bias", False):
        kw["bias"] = 0.2 * torch.randn(n, generator=g, device="cuda")
    compare(lm.route(logits, k, **kw), reference(logits, k, **kw))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("rows", [20, 300])
def test_ties_go_to_the_lowest_index(cuda, score, rows):
    from bafe_b200 import lm
    logits = torch.randint(-2, 3, (rows, 100), generator=gen(3), device="cuda").float()
    for kw in ({}, dict(bias=torch.zeros(100, device="cuda")), dict(groups=10, keep_groups=4),
               dict(bias=torch.zeros(100, device="cuda"), groups=5, keep_groups=2),
               dict(bias=(torch.arange(100, device="cuda") % 2) * 0.25, groups=4, keep_groups=3)):
        compare(lm.route(logits, 9, score=score, **kw), reference(logits, 9, score=score, **kw))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n,groups", [(64, 1), (64, 8), (250, 1), (600, 4)])
def test_near_ties_have_the_order_of_64_bits(cuda, score, n, groups):
    """Biases that make all c equal to within the rounding of the bias: 32-bit scores cannot tell their order."""
    from bafe_b200 import lm
    rows = 150
    logits = torch.randn(1, n, generator=gen(n), device="cuda").expand(rows, n).contiguous()
    logits += 0.001 * torch.randn(rows, 1, generator=gen(n + 1), device="cuda")
    z = logits.double()
    s = torch.softmax(z, -1) if score == "softmax" else torch.sigmoid(z)
    bias = (0.75 - s[0]).float()
    kw = dict(score=score, bias=bias, groups=groups, keep_groups=max(1, groups // 2))
    compare(lm.route(logits, 8, **kw), reference(logits, 8, **kw))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups_whose_worths_are_small_sums_of_large_scores(cuda, score):
    """Worths of some 1e-6 made of scores near 100 and -100: their errors are those of the large ones."""
    from bafe_b200 import lm
    rows, groups = 200, 16
    logits = torch.randn(rows, 2 * groups, generator=gen(4), device="cuda")
    logits[:, 1::2] = logits[:, ::2] + 1e-5 * torch.randn(rows, groups, generator=gen(5), device="cuda")
    bias = torch.empty(2 * groups, device="cuda")
    bias[::2] = 100.0 + torch.arange(groups, device="cuda")
    bias[1::2] = -100.0 - torch.arange(groups, device="cuda")
    s = torch.softmax(logits.double(), -1) if score == "softmax" else torch.sigmoid(logits.double())
    bias[1::2] -= (s[0, ::2] + s[0, 1::2]).float()
    kw = dict(score=score, bias=bias, groups=groups, keep_groups=5)
    compare(lm.route(logits, 6, **kw), reference(logits, 6, **kw))


@pytest.mark.parametrize("rows", [9, 500])
@pytest.mark.parametrize("kw", [dict(), dict(score="sigmoid", renormalize=False), dict(bias=True, groups=4, keep_groups=2)])
def test_shut_experts_and_empty_rows(cuda, rows, kw):
    from bafe_b200 import lm
    g = gen(5)
    kw = dict(kw)
    logits = torch.randn(rows, 40, generator=g, device="cuda")
    logits[torch.rand(rows, 40, generator=g, device="cuda") < 0.5] = -INF
    logits[::3] = -INF
    logits[1::6, 1:] = -INF
    if kw.pop("bias", False):
        kw["bias"] = 0.2 * torch.randn(40, generator=g, device="cuda")
        kw["bias"][7] = -INF
    got = lm.route(logits, 6, **kw)
    compare(got, reference(logits, 6, **kw))
    assert (got.experts[0] == -1).all() and (got.place[0] == -1).all() and (got.weights[0] == 0).all()


def test_lowest_value_masks_and_extremes(cuda):
    """The type's lowest value shuts nothing by itself; far logits keep their order and finite weights."""
    from bafe_b200 import lm
    low = torch.finfo(torch.float32).min
    logits = torch.full((4, 8), low, device="cuda")
    logits[1, 5] = 1.0
    logits[2] = torch.tensor([-300.0, -200, -250, -220, -500, -600, -700, -800], device="cuda")
    logits[3] = torch.tensor([300.0, 200, 250, 220, -500, -600, -700, -800], device="cuda")
    r = lm.route(logits, 3, score="softmax")
    assert r.experts.tolist() == [[0, 1, 2], [5, 0, 1], [1, 3, 2], [0, 2, 3]]
    assert torch.allclose(r.weights[0], torch.full((3,), 1 / 3, device="cuda"))
    assert r.weights[1].tolist() == [1.0, 0.0, 0.0]
    s = lm.route(logits, 3, score="sigmoid")
    assert s.experts.tolist() == r.experts.tolist()
    # scores that underflow still have their ratios: e^-20 and e^-50 of the first
    assert torch.allclose(s.weights[2], torch.tensor([1.0, math.exp(-20), math.exp(-50)], device="cuda"), rtol=1e-5)
    assert torch.allclose(s.weights[3], torch.full((3,), 1 / 3, device="cuda"))


@pytest.mark.parametrize("rows", [3, 300])
def test_nan_rows(cuda, rows):
    from bafe_b200 import lm
    logits = torch.randn(rows, 16, generator=gen(1), device="cuda")
    logits[1, 3] = math.nan
    for score, more in (("softmax", INF), ("sigmoid", math.nan)):
        z = logits.clone()
        z[2, 0] = more
        r = lm.route(z, 4, score=score)
        for t in (1, 2):
            assert r.experts[t].tolist() == [0, 1, 2, 3] and r.weights[t].isnan().all()
        assert not r.weights[0].isnan().any() and int(r.offsets[-1]) == 4 * rows
        assert sorted(r.place.reshape(-1).tolist()) == list(range(4 * rows))


def test_no_rows_and_strided_logits(cuda):
    from bafe_b200 import lm
    r = lm.route(torch.empty(0, 12, device="cuda"), 2)
    assert r.weights.shape == (0, 2) and r.offsets.tolist() == [0] * 13
    wide = torch.randn(90, 41, generator=gen(2), device="cuda")
    a, b = lm.route(wide[:, 3:40], 5), lm.route(wide[:, 3:40].contiguous(), 5)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("rows,n,k", [(20011, 64, 6), (20011, 8, 2), (20011, 300, 9), (16, 256, 8), (17, 256, 8), (64, 33, 5),
                                      (65, 1000, 5), (128, 7, 7), (4737, 129, 3), (37740, 16, 2), (37741, 16, 2),
                                      (90001, 1024, 4), (300000, 5, 1), (150, 256, 31)])
def test_many_rows_place_every_choice(cuda, rows, n, k):
    """Rows over all blocks (and beyond what their counts' bytes hold): places are a permutation sorted by expert,
    equal experts in the choices' order."""
    from bafe_b200 import lm
    logits = torch.randn(rows, n, generator=gen(n), device="cuda")
    logits[torch.rand(rows, generator=gen(n + 1), device="cuda") < 0.1] = -INF
    r = lm.route(logits, k)
    flat, place = r.experts.reshape(-1).long(), r.place.reshape(-1).long()
    some = flat >= 0
    label = torch.where(some, flat, n)
    order = torch.sort(label, stable=True).indices
    want = torch.empty_like(order)
    want[order] = torch.arange(order.numel(), device="cuda")
    assert torch.equal(place[some], want[some]) and (place[~some] == -1).all()
    counts = torch.bincount(label, minlength=n + 1)[:n]
    assert torch.equal(r.offsets.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]))
    again = lm.route(logits, k)
    assert all(torch.equal(a, b) for a, b in zip(r, again))


def test_logits_beyond_32_bit_offsets(cuda):
    """More than 2^31 logits: first and last rows as torch sorts them, and their gradients."""
    from bafe_b200 import lm
    rows, n, k = 2_100_000, 1024, 2
    logits = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    ends = torch.cat([torch.arange(500), torch.arange(rows - 500, rows)]).cuda()
    logits[ends] = torch.randn(1000, n, generator=gen(8), device="cuda").bfloat16()
    logits[500:-500, 7], logits[500:-500, 3] = 2.0, 1.0
    r = lm.route(logits, k)
    order = torch.sort(logits[ends].float(), descending=True, stable=True).indices[:, :k]
    assert torch.equal(r.experts[ends].long(), order)
    middle = r.experts[500:-500]
    assert (middle[:, 0] == 7).all() and (middle[:, 1] == 3).all() and int(r.offsets[-1]) == rows * k
    dw = torch.ones(1, k, device="cuda").expand(rows, k).contiguous()
    dw[:, 1] = -1.0
    dz = lm.route_grad(dw, logits, r.experts, out=logits)
    w = r.weights[ends].double()
    got = dz[ends].gather(1, order).double()
    want = torch.stack([w[:, 0] * (1 - (w[:, 0] - w[:, 1])), w[:, 1] * (-1 - (w[:, 0] - w[:, 1]))], 1)
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14).all()


def grad64(dw, logits, experts, score, renormalize, scale):
    z = logits.double().requires_grad_()
    p = torch.softmax(z, -1) if score == "softmax" else torch.sigmoid(z)
    inside = (experts >= 0) & (experts < z.shape[1])
    w = p.gather(1, experts.long().clamp(0, z.shape[1] - 1)) * inside
    if renormalize:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
    g = dw.double() * scale * inside
    dz = torch.autograd.grad((w * g).sum(), z)[0]
    size = torch.zeros_like(dz).scatter_add_(1, experts.long().clamp(0, z.shape[1] - 1), w.detach().abs() * g.abs())
    if not renormalize and score == "softmax":
        size = size + p.detach() * (w.detach().abs() * g.abs()).sum(-1, keepdim=True)
    elif renormalize:
        size = size + torch.zeros_like(dz).scatter_add_(1, experts.long().clamp(0, z.shape[1] - 1), w.detach().abs() * inside) \
            * (w.detach().abs() * g.abs()).sum(-1, keepdim=True)
    # what cancels in exact arithmetic leaves torch's own 64-bit rounding: some 32 of 2^-53 of the row's largest terms
    return dz, size + 2.0 ** -48 / (2 * REL) * g.abs().sum(-1, keepdim=True)


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (5, 8, 2), (300, 60, 4), (77, 256, 8), (33, 1024, 31)])
@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradient(cuda, rows, n, k, score, renormalize, dtype):
    from bafe_b200 import lm
    g = gen(rows + n)
    logits = (2.0 * torch.randn(rows, n, generator=g, device="cuda")).to(dtype)
    experts = torch.rand(rows, n, generator=g, device="cuda").topk(k, -1).indices.int()
    if k > 1:
        experts[::2, k // 2] = -1
    dw = torch.randn(rows, k, generator=g, device="cuda")
    got = lm.route_grad(dw, logits, experts, score=score, renormalize=renormalize, scale=1.5)
    want, size = grad64(dw, logits, experts, score, renormalize, 1.5)
    assert got.dtype == dtype
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    bound = 2 * REL * size + torch.finfo(dtype).eps / 2 * want.abs() + tiny
    assert ((got.double() - want).abs() <= bound).all()
    # in place of the logits, and with one row of gradients for all
    one = dw[:1].expand(rows, k)
    want2 = lm.route_grad(one.contiguous(), logits, experts, score=score, renormalize=renormalize)
    held = logits.clone()
    assert lm.route_grad(one, held, experts, score=score, renormalize=renormalize, out=held) is held
    assert torch.equal(held, want2)


@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_gradient_against_differences(cuda, score, renormalize):
    """(w(z + h) - w(z - h)) / 2h of the forward call's own weights.  h = 2^-6: the difference is off by h^2 / 6 times
    the third derivative (below 1) and by the weights' errors, 2 * 2^-17 / 2h: 2^-14.6 + 2^-11 in all per choice."""
    from bafe_b200 import lm
    z = torch.randn(1, 12, generator=gen(9), device="cuda").mul(64).round().div(64)
    z[0, :4] += 3.0                                      # the choice stays the same
    kw = dict(score=score, renormalize=renormalize)
    r = lm.route(z, 4, **kw)
    dw = torch.tensor([[0.5, -1.0, 0.25, 1.0]], device="cuda")
    got = lm.route_grad(dw, z, r.experts, **kw)
    h = 2.0 ** -6
    for i in range(12):
        side = []
        for sign in (h, -h):
            v = z.clone()
            v[0, i] += sign
            q = lm.route(v, 4, **kw)
            w = torch.zeros(12, device="cuda").index_put_((q.experts[0].long(),), q.weights[0])
            side.append(w[r.experts[0].long()].double())
        slope = float(((side[0] - side[1]) / (2 * h) * dw[0].double()).sum())
        assert abs(slope - float(got[0, i])) <= 4 * (2.0 ** -14.6 + 2.0 ** -11)


def test_refusals(cuda):
    from bafe_b200 import lm
    z = torch.randn(4, 16, device="cuda")
    for bad in (dict(k=0), dict(k=17), dict(k=4, score="tanh"), dict(k=4, groups=3), dict(k=4, groups=0),
                dict(k=4, groups=4, keep_groups=5), dict(k=9, groups=4, keep_groups=2), dict(k=4, group_top=3),
                dict(k=4, keep_groups=2), dict(k=4, bias=torch.zeros(15, device="cuda")),
                dict(k=4, bias=torch.zeros(16, device="cuda", dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            lm.route(z, **bad)
    with pytest.raises(TypeError):
        lm.route(z.double(), 2)
    with pytest.raises(TypeError):
        lm.route(z, 2.0)
    with pytest.raises(ValueError):
        lm.route(torch.randn(2, 1025, device="cuda"), 2)
    with pytest.raises(ValueError, match="gradient"):
        lm.route(z.clone().requires_grad_(), 2)
    with pytest.raises(RuntimeError):
        lm.route(z, 2, scale=INF)
    e, d = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")
    for bad in ((d, z, e.long()), (d[:, :1], z, e), (d.half(), z, e), (d[:3], z, e), (d, z, e[:1].expand(4, 2)),
                (torch.zeros(4, 17, device="cuda"), z, torch.zeros(4, 17, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            lm.route_grad(*bad)
    with pytest.raises(ValueError):
        lm.route_grad(d, z, e, out=torch.empty(4, 15, device="cuda"))
