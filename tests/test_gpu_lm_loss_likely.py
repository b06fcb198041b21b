"""Cross entropy of rows whose target is likely: there the gradient is dloss
times 1 - p, which is small, and the logits that the gradient computes have to
be those that lse was made of.

Bounds.  The tensor core truncates, so a logit made of products of one sign
comes out short by some 1e-6 of itself; where both passes are short alike,
p = exp(z - lse) is that of logits scaled by as much, and 1 - p is off by some
1e-5 of itself.  What remains is the sum of exponentials (below 2^-20 of it, as
in test_gpu_lm_loss.py), lse's rounding (half a step, 2^-20 below 32) and the
exponential's own 2^-22: the target's entry of g is off by less than
DELTA = 2^-19 + 2^-21 of dloss, which its column of w (row of x) carries into
dx (dw).  The roundings of g and of the result count as in test_gpu_lm_loss.py.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}      # 2-norm of a rounding: u / sqrt(3), rounded up
DELTA = 2.0 ** -19 + 2.0 ** -21


@pytest.mark.parametrize("rows,vocab,width", [(40, 8000, 4096), (128, 8000, 4096), (300, 8000, 4096), (300, 8000, 2056)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_likely_targets(cuda, rows, vocab, width, dtype):
    from bafe_b200 import lm
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    w = torch.randn(vocab, width, generator=g, device="cuda").to(dtype)
    target = torch.randperm(vocab, generator=g, device="cuda")[:rows]
    # hidden states along their target's weights: its logit is 14 to 18, a sum of terms of one sign, the others about 0
    size = torch.linspace(14.0, 18.0, rows, device="cuda") / w[target].float().square().sum(-1)
    x = (w[target].float() * size[:, None] * 64).to(dtype)         # and w a 64th: f16 keeps x's bits
    w = w / 64
    dloss = torch.ones(rows, device="cuda")
    loss, lse = lm.linear_cross_entropy(x, w, target)
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    x64, w64 = x.double(), w.double()
    z = x64 @ w64.t()
    own = z[torch.arange(rows), target]
    assert (z.argmax(-1) == target).all() and 13.5 < float(own.min()) and float(own.max()) < 18.5
    gr = torch.softmax(z, -1)
    miss = (torch.exp(z - own[:, None]).sum(-1) - 1.0) / torch.exp(z - own[:, None]).sum(-1)
    gr[torch.arange(rows), target] = -miss                         # p - 1 without cancelling
    assert 1e-5 < float(miss.min()) and float(miss.min()) < 2e-4
    want = gr @ w64
    bound = DELTA * w64[target].norm(dim=-1) + 2 * 2 ** 0.5 * HALF[dtype] * want.norm(dim=-1)
    off = (dx.double() - want).norm(dim=-1)
    assert (off <= bound).all(), float((off / bound).max())
    want = (gr.t() @ x64)[target]
    bound = DELTA * x64.norm(dim=-1) + 2 * 2 ** 0.5 * HALF[dtype] * want.norm(dim=-1)
    off = (dw[target].double() - want).norm(dim=-1)
    assert (off <= bound).all(), float((off / bound).max())


def test_one_word(cuda):
    """A vocabulary of one word: p is 1, nothing has a gradient."""
    from bafe_b200 import lm
    for rows in (5, 200):
        x = torch.randn(rows, 512, device="cuda").bfloat16()
        w = torch.randn(1, 512, device="cuda").bfloat16()
        t = torch.zeros(rows, dtype=torch.int64, device="cuda")
        loss, lse = lm.linear_cross_entropy(x, w, t)
        # p - 1 = expm1(z - lse): lse's rounding, half a step of |z| < 128, and its sum's, 2^-20
        limit = 2.0 ** -18 + 2.0 ** -20
        assert float(lse.abs().max()) < 128
        dx, _ = lm.linear_cross_entropy_grad(torch.ones(rows, device="cuda"), x, w, t, lse)
        assert (dx.double().abs() <= limit * w.double().abs() * (1 + 2.0 ** -7)).all()
