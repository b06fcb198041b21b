"""The order of routed experts where scores saturate, underflow or biases are
very large (lm.route): without a bias it is that of the logits, which goes on
where scores are equal; with one that of score + bias in 64 bits, the lower
index of equals."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_saturated_scores(cuda, rows):
    """Sigmoid scores above 37 are 1 in 64 bits: the larger logit without a bias, the lower index with one of zeros."""
    from bafe_b200 import lm
    n, k = 64, 4
    logits = 38.0 + 40.0 * torch.rand(rows, n, generator=gen(rows), device="cuda")
    by_logit = torch.sort(logits, descending=True, stable=True).indices[:, :k].int()
    zeros = torch.zeros(n, device="cuda")
    first = torch.arange(k, device="cuda", dtype=torch.int32).expand(rows, k)
    assert torch.equal(lm.route(logits, k, score="sigmoid").experts, by_logit)
    assert torch.equal(lm.route(logits, k, score="sigmoid", bias=zeros).experts, first)
    # groups of equal worth: the lowest stay, and in them the logits' order without a bias
    kept = torch.sort(logits[:, :32], descending=True, stable=True).indices[:, :k].int()
    for keep, want in ((4, kept), (8, by_logit)):
        assert torch.equal(lm.route(logits, k, score="sigmoid", groups=8, keep_groups=keep).experts, want)
    for keep in (4, 8):
        assert torch.equal(lm.route(logits, k, score="sigmoid", bias=zeros, groups=8, keep_groups=keep).experts, first)


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_that_underflow(cuda, rows, score):
    """Scores below e^-700 count as 0 beside a bias, and keep the logits' order without one."""
    from bafe_b200 import lm
    n, k = 16, 5
    logits = torch.full((rows, n), -1000.0, device="cuda")
    logits += 50.0 * torch.rand(rows, n, generator=gen(rows), device="cuda")          # -1000 to -950
    logits[:, 9] = 0.0
    by_logit = torch.sort(logits, descending=True, stable=True).indices[:, :k].int()
    assert torch.equal(lm.route(logits, k, score=score).experts, by_logit)
    got = lm.route(logits, k, score=score, bias=torch.zeros(n, device="cuda")).experts
    assert torch.equal(got, torch.tensor([9, 0, 1, 2, 3], dtype=torch.int32, device="cuda").expand(rows, k))


@pytest.mark.parametrize("rows", [3, 40, 300])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_groups_whose_worth_leaves_the_range_of_32_bits(cuda, rows, score, sign):
    """Two biases of 2e38 and more are beyond f32: the groups' worths differ all the same."""
    from bafe_b200 import lm
    n, groups, keep, k = 48, 12, 5, 6
    size = n // groups
    logits = torch.randn(rows, n, generator=gen(rows), device="cuda")
    order = torch.randperm(n, generator=gen(1), device="cuda").float()
    bias = sign * (2.0e38 + 1.0e36 * order)              # finite, all different by more than any score
    if sign < 0:
        logits[:, 4:8] = -math.inf                       # a shut group is worth less than any of an open one
    c = torch.sigmoid(logits.double()) if score == "sigmoid" else torch.softmax(logits.double(), -1)
    c = torch.where(logits > -math.inf, c + bias.double(), -math.inf)
    worth = c.view(rows, groups, size).sort(-1, descending=True).values[..., :2].sum(-1)
    stay = torch.sort(worth, dim=-1, descending=True, stable=True).indices[:, :keep]
    open_ = torch.zeros(rows, groups, dtype=torch.bool, device="cuda").scatter_(1, stay, True).repeat_interleave(size, 1)
    want = torch.sort(torch.where(open_, c, -math.inf), dim=-1, descending=True, stable=True).indices[:, :k].int()
    got = lm.route(logits, k, score=score, bias=bias, groups=groups, keep_groups=keep)
    assert torch.equal(got.experts, want)
