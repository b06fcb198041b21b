"""Rows of the cross entropy that count for nothing, or differ from one
another in size or kind, on every kernel that computes it: up to 128 rows, more
of them, and more than 8192, whose common factor a kernel of its own finds."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS = [40, 300, 9000]
TYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(rows, dtype, vocab=300, width=64, size=2.0):
    x = torch.randn(rows, width, generator=gen(rows), device="cuda").to(dtype)
    w = (torch.randn(vocab, width, generator=gen(7), device="cuda") * (size / math.sqrt(width))).to(dtype)
    target = torch.randint(0, vocab, (rows,), generator=gen(9), device="cuda")
    return x, w, target


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
def test_losses_of_ignored_rows_change_no_bit(cuda, rows, dtype):
    """However large, infinite or NaN: the gradients are those with 0 there."""
    from bafe_b200 import lm
    x, w, target = make(rows, dtype)
    target[torch.rand(rows, generator=gen(1), device="cuda") < 0.2] = -100
    target[1] = -100
    ignored = target == -100
    dloss = 1e-3 * torch.randn(rows, generator=gen(2), device="cuda")
    _, lse = lm.linear_cross_entropy(x, w, target)
    want = lm.linear_cross_entropy_grad(torch.where(ignored, 0.0, dloss), x, w, target, lse)
    assert float(want[0].abs().max()) > 1e-5 and float(want[1].abs().max()) > 1e-5
    for factor in (1.0, 1e3, 1e9, 1e27, 1e38, math.inf, math.nan):
        got = lm.linear_cross_entropy_grad(torch.where(ignored, factor, dloss), x, w, target, lse)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), factor
    got = lm.linear_cross_entropy_grad(torch.where(ignored, 1e20, dloss), x, w, target.int(), lse)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
def test_losses_of_rows_out_of_range_change_no_other_row(cuda, rows, dtype):
    from bafe_b200 import lm
    x, w, target = make(rows, dtype)
    target[3], target[rows - 1] = 300, -7
    counted = (target >= 0) & (target < 300)
    dloss = 1e-3 * torch.randn(rows, generator=gen(2), device="cuda")
    _, lse = lm.linear_cross_entropy(x, w, target)
    want, _ = lm.linear_cross_entropy_grad(torch.where(counted, dloss, 0.0), x, w, target, lse)
    assert want[~counted].isnan().all() and not want[counted].isnan().any()
    for factor in (1e9, 1e38, math.inf):
        got, dw = lm.linear_cross_entropy_grad(torch.where(counted, dloss, factor), x, w, target, lse)
        assert torch.equal(got[counted], want[counted]) and got[~counted].isnan().all() and dw.isnan().all()


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
def test_targets(cuda, rows, dtype):
    """Ignored rows add nothing whatever lse says; an index of the vocabulary may be ignored; all rows may be."""
    from bafe_b200 import lm
    x, w, target = make(rows, dtype)
    target[3], target[7] = -100, 0
    dloss = torch.randn(rows, generator=gen(2), device="cuda") / rows
    loss, lse = lm.linear_cross_entropy(x, w, target)
    assert loss[3] == 0 and not loss.isnan().any()
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    for value in (math.nan, math.inf, -math.inf):
        held = lse.clone()
        held[3] = value
        again = lm.linear_cross_entropy_grad(dloss, x, w, target, held)
        assert (again[0][3] == 0).all() and torch.equal(again[0], dx) and torch.equal(again[1], dw)
    # ignoring word 0 is ignoring the rows that want it
    moved = torch.where(target == 0, -100, target)
    moved_loss, _ = lm.linear_cross_entropy(x, w, moved)
    want = lm.linear_cross_entropy_grad(dloss, x, w, moved, lse)
    here = torch.where(target == -100, 0, target)
    here_loss, _ = lm.linear_cross_entropy(x, w, here, ignore_index=0)
    got = lm.linear_cross_entropy_grad(dloss, x, w, here, lse, ignore_index=0)
    assert torch.equal(here_loss, moved_loss) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    none = torch.full_like(target, -100)
    loss, lse2 = lm.linear_cross_entropy(x, w, none)
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, none, lse2)
    assert torch.equal(lse2, lse) and (loss == 0).all() and (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("rows", ROWS)
def test_extreme_logits(cuda, rows):
    """Logits in the thousands, a row of equal ones, infinities and NaN in one row only."""
    from bafe_b200 import lm
    x, w, target = make(rows, torch.bfloat16, vocab=500, size=2000.0)
    x[1] = 0
    dloss = torch.ones(rows, device="cuda") / rows
    loss, lse = lm.linear_cross_entropy(x, w, target)
    assert abs(float(loss[1]) - math.log(500)) < 1e-5
    want = torch.logsumexp(x.double() @ w.double().t(), -1)
    assert float(((lse.double() - want).abs() / (1 + want.abs())).max()) < 2.0 ** -18
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    assert not dx.isnan().any() and not dw.isnan().any()
    x[2, 3], x[3, 0] = math.nan, math.inf
    loss2, _ = lm.linear_cross_entropy(x, w, target)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[2:4] = True
    assert loss2[bad].isnan().all() and torch.equal(loss2[~bad], loss[~bad])


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
def test_losses_gradients_of_all_sizes(cuda, rows, dtype):
    """Powers of two in dloss come out again bit for bit (where the results stay in the type's normal range), one value
    for all rows is that value in each, and zeros give zeros."""
    from bafe_b200 import lm
    x, w, target = make(rows, dtype)
    w = w / 16
    _, lse = lm.linear_cross_entropy(x, w, target)
    one = torch.ones(1, device="cuda").expand(rows)
    want = lm.linear_cross_entropy_grad(one, x, w, target, lse)
    same = lm.linear_cross_entropy_grad(one.contiguous(), x, w, target, lse)
    assert torch.equal(same[0], want[0]) and torch.equal(same[1], want[1])
    for power in ((4, -3) if dtype == torch.float16 else (20, -30, 90)):
        got = lm.linear_cross_entropy_grad(one * 2.0 ** power, x, w, target, lse)
        for a, b in zip(got, want):
            fine = (b.double().abs() > 2.0 ** -10) & (b.double().abs() < 2.0 ** 10)
            assert int(fine.sum()) > b.numel() // 8
            assert torch.equal(a.double()[fine], b.double()[fine] * 2.0 ** power)
    zero = lm.linear_cross_entropy_grad(0 * one, x, w, target, lse)
    assert (zero[0] == 0).all() and (zero[1] == 0).all()
