"""Cross entropy from hidden states and output weights (lm.linear_cross_entropy
and its gradient) against the definition in 64 bits.

Bounds.  A logit is summed on the tensor cores, 16 products an instruction,
each adding at most 2^-22 of the sum of sizes S = sum |x w|: its error is below
(width / 16 + 1) 2^-22 S.  The sum of exponentials adds roundings of 2^-22 to
2^-24 each, below 2^-20 of it in all, and lse is rounded (2^-23 |lse|).
g = dloss (p - onehot) carries the logit's and lse's error in p, and one
rounding u = half a step of the type; dx and dw carry the errors of g through
their sums (all signs alike: an upper bound), add up as the logits do, and
are rounded once more.  In the 2-norm the roundings are independent: u / sqrt(3)
each, g's and the result's, twice as much allowed.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}      # 2-norm of a rounding: u / sqrt(3), rounded up


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(rows, vocab, width, dtype, seed=0, ignored=0.1, size=2.0):
    g = gen(seed + rows + 3 * vocab + 7 * width)
    x = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    w = (torch.randn(vocab, width, generator=g, device="cuda") * (size / math.sqrt(width))).to(dtype)
    target = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    if rows > 1:
        target[torch.rand(rows, generator=g, device="cuda") < ignored] = -100
    dloss = torch.randn(rows, generator=g, device="cuda") / rows
    return x, w, target, dloss


def reference(x, w, target, dloss, ignore=-100):
    x, w = x.double(), w.double()
    z = x @ w.t()
    lse = torch.logsumexp(z, -1)
    counts = target != ignore
    at = torch.where(counts, target, 0).long()
    loss = torch.where(counts, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    p = torch.exp(z - lse[:, None])
    scale = dloss.double() * counts
    g = p.clone()
    g.scatter_add_(1, at[:, None], -torch.ones_like(at, dtype=torch.float64)[:, None])
    g *= scale[:, None]
    return z, lse, loss, p, scale, g


def check(x, w, target, dloss, got, ignore=-100):
    """Both calls' results within the bounds, element by element, and the gradients' 2-norms."""
    loss, lse, dx, dw = got
    z, lse64, loss64, p, scale, g = reference(x, w, target, dloss, ignore)
    width, vocab, rows, u = x.shape[1], w.shape[0], x.shape[0], torch.finfo(x.dtype).eps / 2
    ax, aw = x.double().abs(), w.double().abs()
    zerr = (width / 16 + 1) * 2.0 ** -22 * (ax @ aw.t()).amax(-1)
    lerr = zerr + 2.0 ** -20 + 2.0 ** -23 * lse64.abs()
    assert ((lse.double() - lse64).abs() <= lerr).all(), float(((lse.double() - lse64).abs() / lerr).max())
    assert ((loss.double() - loss64).abs() <= lerr + zerr + 2.0 ** -23 * z.abs().amax(-1)).all()
    gerr = p * (scale.abs() * (zerr + lerr + 2.0 ** -19))[:, None] + u * g.abs()
    if x.dtype == torch.float16:
        gerr = gerr + dloss.double().abs().max() * 2.0 ** -36      # g's smallest numbers, scaled
    for name, have, want, err, n, size in (
            ("dx", dx, g @ w.double(), gerr @ aw, vocab, g.abs() @ aw),
            ("dw", dw, g.t() @ x.double(), gerr.t() @ ax, rows, g.t().abs() @ ax)):
        tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-38
        bound = err + (n / 16 + 2) * 2.0 ** -22 * size + u * want.abs() * (1 + u) + tiny
        if x.dtype == torch.float16:                     # what leaves f16's range is infinite
            assert (have[want.abs() - bound >= 65520.0].isinf()).all(), name
            inside = want.abs() + bound < 65504.0
            have, want, bound = have[inside], want[inside], bound[inside]
        off = (have.double() - want).abs()
        assert (off <= bound).all(), (name, float((off / bound).max()))
        if want.numel() >= 4096 and (x.dtype != torch.float16 or float(want.abs().mean()) > 2.0 ** -14):
            assert float(off.norm() / want.norm()) < 2 * 2 ** 0.5 * HALF[x.dtype], name


def both(lm, x, w, target, dloss, **kw):
    loss, lse = lm.linear_cross_entropy(x, w, target, **kw)
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, target, lse, **kw)
    return loss, lse, dx, dw


@pytest.mark.parametrize("rows,vocab,width", [
    (1, 1, 1), (1, 2, 8), (2, 63, 16), (3, 64, 64), (31, 65, 63), (127, 255, 72), (128, 256, 128), (129, 257, 65),
    (256, 512, 256), (257, 1000, 200), (600, 5003, 264), (1000, 300, 1150), (5, 40000, 520), (2100, 2050, 40),
    (16, 8192, 1024), (300, 20000, 64), (33, 3000, 130), (96, 1111, 200), (130, 2500, 320), (160, 777, 96), (224, 300, 2056),
    (225, 300, 136), (450, 6000, 72), (777, 4001, 88), (17, 130, 4096), (1300, 513, 1040),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_loss_and_gradient(cuda, rows, vocab, width, dtype):
    from bafe_b200 import lm
    x, w, target, dloss = make(rows, vocab, width, dtype)
    check(x, w, target, dloss, both(lm, x, w, target, dloss))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab,width", [(70000, 8500, 24), (300, 1000003, 24), (100, 3000017, 16)])
def test_gradient_in_pieces(cuda, rows, vocab, width, dtype):
    """g of more than one piece (of some 4000 to 1500000 words), dx summed over them."""
    from bafe_b200 import lm
    x, w, target, dloss = make(rows, vocab, width, dtype)
    loss, lse = lm.linear_cross_entropy(x, w, target)
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    total = torch.zeros(vocab, width, dtype=torch.float64, device="cuda")
    part = 10000 if rows > 1000 else 100
    for a in range(0, rows, part):
        s = slice(a, a + part)
        z, lse64, loss64, p, scale, g = reference(x[s], w, target[s], dloss[s])
        assert float((lse[s].double() - lse64).abs().max()) < 2.0 ** -16 and float((loss[s].double() - loss64).abs().max()) < 2.0 ** -15
        want = g @ w.double()
        if dtype == torch.bfloat16 or rows < 1000:       # f16 results of 1 / 70000 are among its smallest numbers
            assert float((dx[s].double() - want).norm() / want.norm()) < 2 * 2 ** 0.5 * HALF[dtype]
        else:
            assert float((dx[s].double() - want).abs().max()) < 2.0 ** -24
        total += g.t() @ x[s].double()
    assert float((dw.double() - total).norm() / total.norm()) < 2 * 2 ** 0.5 * HALF[dtype]
    again = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("offset,extra", [(0, 8), (1, 0), (3, 5), (8, 16), (0, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_strides_and_offsets(cuda, offset, extra, dtype):
    from bafe_b200 import lm
    rows, vocab, width = 200, 700, 96

    def inside(n, values=None):
        buf = torch.full((n * (width + extra) + offset,), 7.0, dtype=dtype, device="cuda")
        t = torch.as_strided(buf, (n, width), (width + extra, 1), offset)
        if values is not None:
            t.copy_(values)
        return buf, t

    x, w, target, dloss = make(rows, vocab, width, dtype)
    want = both(lm, x, w, target, dloss)
    _, xs = inside(rows, x)
    _, ws = inside(vocab, w)
    loss, lse = lm.linear_cross_entropy(xs, ws, target.int())
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    bx, ox = inside(rows)
    bw, ow = inside(vocab)
    dx, dw = lm.linear_cross_entropy_grad(dloss, xs, ws, target.int(), lse, out=ox, weight_out=ow)
    assert dx is ox and dw is ow and torch.equal(dx, want[2]) and torch.equal(dw, want[3])
    ox.fill_(7.0), ow.fill_(7.0)
    assert (bx == 7.0).all() and (bw == 7.0).all()       # nothing beside the rows was written


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_targets(cuda, dtype):
    """Ignored rows add nothing whatever lse says; rows out of range give NaN; an index of the vocabulary may be ignored."""
    from bafe_b200 import lm
    x, w, target, dloss = make(40, 300, 64, dtype, ignored=0.0)
    target[3], target[7] = -100, 0
    target[target == 299] = 5
    loss, lse = lm.linear_cross_entropy(x, w, target)
    assert loss[3] == 0 and not loss.isnan().any()
    held = lse.clone()
    held[3] = math.nan
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, target, held)
    assert (dx[3] == 0).all()
    check(x, w, target, dloss, (loss, lse, dx, dw))
    other = torch.where(target == -100, 1, target)
    check(x, w, other, dloss, both(lm, x, w, other, dloss, ignore_index=0), ignore=0)
    for bad in (300, -1, 1 << 40):
        t = target.clone()
        t[5] = bad
        loss, lse2 = lm.linear_cross_entropy(x, w, t)
        assert loss[5].isnan() and not loss[:5].isnan().any() and torch.equal(lse, lse2)
        dx, _ = lm.linear_cross_entropy_grad(dloss, x, w, t, lse)
        assert dx[5].isnan().all() and not dx[:5].isnan().any()
    none = torch.full_like(target, -100)
    loss, lse = lm.linear_cross_entropy(x, w, none)
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, none, lse)
    assert (loss == 0).all() and (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [2.0 ** -30, 1.0, 2.0 ** 20])
def test_losses_gradients_of_all_sizes(cuda, dtype, size):
    """dloss far from 1, and one value for all rows (stride 0)."""
    from bafe_b200 import lm
    x, w, target, _ = make(150, 400, 80, dtype)
    x = x * (2.0 ** -4 if size > 1 else 1.0)
    dloss = torch.full((1,), size / 16, device="cuda").expand(150)
    loss, lse = lm.linear_cross_entropy(x, w, target)
    got = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    same = lm.linear_cross_entropy_grad(dloss.contiguous(), x, w, target, lse)
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])
    check(x, w, target, dloss, (loss, lse) + got)
    zero = lm.linear_cross_entropy_grad(torch.zeros(150, device="cuda"), x, w, target, lse)
    assert (zero[0] == 0).all() and (zero[1] == 0).all()


def test_extreme_logits(cuda):
    """Logits in the thousands, a row of equal ones, infinities and NaN in one row only."""
    from bafe_b200 import lm
    x, w, target, dloss = make(64, 500, 64, torch.bfloat16, size=2000.0, ignored=0.0)
    x[1] = 0
    got = both(lm, x, w, target, dloss)
    assert abs(float(got[0][1]) - math.log(500)) < 1e-5
    z = x.double() @ w.double().t()
    lse = torch.logsumexp(z, -1)
    assert float(((got[1].double() - lse).abs() / (1 + lse.abs())).max()) < 2.0 ** -18
    assert not got[2].isnan().any() and not got[3].isnan().any()
    x[2, 3], x[3, 0] = math.nan, math.inf
    loss, lse2 = lm.linear_cross_entropy(x, w, target)
    bad = torch.zeros(64, dtype=torch.bool, device="cuda")
    bad[2:4] = True
    assert loss[bad].isnan().all() and torch.equal(loss[~bad], got[0][~bad])


def test_gradient_against_differences(cuda):
    """(loss(x + h) - loss(x - h)) / 2h with h = 2^-5, exact in f16.  The third derivative along a weight column of
    sizes up to 1 is below 8; the difference is off by 8 h^2 / 6 < 2^-9.5, f32 losses of about 4 by 2^-21 / h = 2^-16,
    the gradient by its roundings, 2^-10 of sums of sizes up to 2."""
    from bafe_b200 import lm
    rows, vocab, width = 3, 50, 16
    x = torch.randn(rows, width, generator=gen(1), device="cuda").mul(32).round().div(32).half()
    w = torch.rand(vocab, width, generator=gen(2), device="cuda").mul(2).sub(1).mul(32).round().div(32).half()
    target = torch.tensor([4, 49, 0], device="cuda")
    _, lse = lm.linear_cross_entropy(x, w, target)
    dx, dw = lm.linear_cross_entropy_grad(torch.ones(rows, device="cuda"), x, w, target, lse)
    h = 2.0 ** -5
    limit = 2.0 ** -9.5 + 2.0 ** -16 + 2.0 ** -9

    def total(a, b):
        return float(lm.linear_cross_entropy(a, b, target)[0].double().sum())

    for i, j in ((0, 0), (1, 7), (2, 15)):
        a, b = x.clone(), x.clone()
        a[i, j] += h
        b[i, j] -= h
        assert abs((total(a, w) - total(b, w)) / (2 * h) - float(dx[i, j])) < limit
    x = x / 4                                            # along w the derivatives are x's powers: below 8 as well
    _, lse = lm.linear_cross_entropy(x, w, target)
    _, dw = lm.linear_cross_entropy_grad(torch.ones(rows, device="cuda"), x, w, target, lse)
    for i, j in ((0, 0), (4, 3), (49, 15), (20, 8)):
        a, b = w.clone(), w.clone()
        a[i, j] += h
        b[i, j] -= h
        assert abs((total(x, a) - total(x, b)) / (2 * h) - float(dw[i, j])) < limit


def test_weights_beyond_32_bit_offsets(cuda):
    """Weights, and their gradient, of more than 2^31 elements."""
    from bafe_b200 import lm
    rows, vocab, width = 2, 1049000, 2056
    w = torch.empty(vocab, width, dtype=torch.bfloat16, device="cuda")
    w.normal_(0.0, 0.02, generator=gen(1))
    x = torch.randn(rows, width, generator=gen(2), device="cuda").bfloat16()
    target = torch.tensor([vocab - 1, 3], device="cuda")
    dloss = torch.ones(rows, device="cuda")
    loss, lse = lm.linear_cross_entropy(x, w, target)
    z = torch.cat([x.double() @ w[a:a + 65536].double().t() for a in range(0, vocab, 65536)], 1)
    lse64 = torch.logsumexp(z, -1)
    assert float((lse.double() - lse64).abs().max()) < 1e-4
    assert float((loss.double() - (lse64 - z[torch.arange(2), target])).abs().max()) < 2e-4
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    g = torch.exp(z - lse64[:, None])
    g[torch.arange(2), target] -= 1.0
    for a in (0, 1 << 19, (1 << 20) - 256, vocab - 300):
        want = g[:, a:a + 300].t() @ x.double()
        assert float((dw[a:a + 300].double() - want).norm() / want.norm()) < 2 * 2 ** 0.5 * HALF[torch.bfloat16]
    want = sum(g[:, a:a + 65536] @ w[a:a + 65536].double() for a in range(0, vocab, 65536))
    assert float((dx.double() - want).norm() / want.norm()) < 2 * 2 ** 0.5 * HALF[torch.bfloat16]


def test_rows_beyond_32_bit_offsets(cuda):
    """Hidden states, and their gradient, of more than 2^31 elements."""
    from bafe_b200 import lm
    rows, vocab, width = 525000, 260, 4104
    x = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    x.normal_(0.0, 1.0, generator=gen(1))
    w = (torch.randn(vocab, width, generator=gen(2), device="cuda") * (2.0 / math.sqrt(width))).bfloat16()
    target = torch.randint(0, vocab, (rows,), generator=gen(3), device="cuda")
    dloss = torch.ones(rows, device="cuda")
    loss, lse = lm.linear_cross_entropy(x, w, target)
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    for s in (slice(0, 400), slice(rows // 2, rows // 2 + 400), slice(rows - 400, rows)):
        _, lse64, loss64, _, _, g = reference(x[s], w, target[s], dloss[s])
        assert float((lse[s].double() - lse64).abs().max()) < 1e-4 and float((loss[s].double() - loss64).abs().max()) < 2e-4
        want = g @ w.double()
        assert float((dx[s].double() - want).norm() / want.norm()) < 2 * 2 ** 0.5 * HALF[torch.bfloat16]
    total = torch.zeros(vocab, width, dtype=torch.float64, device="cuda")
    for a in range(0, rows, 25000):
        s = slice(a, a + 25000)
        total += reference(x[s], w, target[s], dloss[s])[5].t() @ x[s].double()
    assert float((dw.double() - total).norm() / total.norm()) < 2 * 2 ** 0.5 * HALF[torch.bfloat16]


def test_empty_calls(cuda):
    from bafe_b200 import lm
    x, w, t = torch.empty(0, 64, device="cuda").bfloat16(), torch.randn(30, 64, device="cuda").bfloat16(), torch.empty(0, dtype=torch.int64, device="cuda")
    loss, lse = lm.linear_cross_entropy(x, w, t)
    assert loss.shape == lse.shape == (0,)
    dx, dw = lm.linear_cross_entropy_grad(loss, x, w, t, lse)
    assert dx.shape == (0, 64) and dw.shape == (30, 64) and (dw == 0).all()


def test_refusals(cuda):
    from bafe_b200 import lm
    x, w, target, dloss = make(8, 50, 64, torch.bfloat16)
    lse = torch.zeros(8, device="cuda")
    for call in (lambda: lm.linear_cross_entropy(x, w.half(), target), lambda: lm.linear_cross_entropy(x, w[:, :63], target),
                 lambda: lm.linear_cross_entropy(x, w, target[:7]), lambda: lm.linear_cross_entropy(x, w, target.float()),
                 lambda: lm.linear_cross_entropy(x, w, target[:, None]), lambda: lm.linear_cross_entropy(x, w[:0], target),
                 lambda: lm.linear_cross_entropy(x, w.t().contiguous().t(), target),
                 lambda: lm.linear_cross_entropy(x.cpu(), w, target), lambda: lm.linear_cross_entropy(x, w, target.cpu()),
                 lambda: lm.linear_cross_entropy(x.clone().requires_grad_(), w, target),
                 lambda: lm.linear_cross_entropy_grad(dloss.half(), x, w, target, lse),
                 lambda: lm.linear_cross_entropy_grad(dloss[:7], x, w, target, lse),
                 lambda: lm.linear_cross_entropy_grad(dloss, x, w, target, lse[:7]),
                 lambda: lm.linear_cross_entropy_grad(dloss, x, w, target, lse, out=x),
                 lambda: lm.linear_cross_entropy_grad(dloss, x, w, target, lse, weight_out=w),
                 lambda: lm.linear_cross_entropy_grad(dloss, x, w, target, lse, out=torch.empty(8, 65, device="cuda").bfloat16())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        lm.linear_cross_entropy(x.float(), w.float(), target)
    with pytest.raises(TypeError):
        lm.linear_cross_entropy(x, w, target, ignore_index=1.5)
    with pytest.raises(ValueError):
        lm.linear_cross_entropy(x, w, target, ignore_index=(1 << 64) - 100)
