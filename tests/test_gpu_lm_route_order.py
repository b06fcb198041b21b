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
