"""The cross entropy's gradient of rows with very different dloss, and
over very many rows or words."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("rows", [100, 250])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_of_different_losses(cuda, rows, dtype):
    """dloss from 1 to 2^-24 of the largest, row by row, with a loss scale that keeps dx in f16's normal range.

    g is dloss q with q = p - onehot, rounded to the type: half a step u relative, and in f16, where the largest dloss
    is 2^15, 2^-25 at the least, 2^-40 of the largest dloss.  These roundings are independent (u / sqrt(3) and
    2^-40 / sqrt(3)): in the 2-norm they come to sqrt(sum_v (u^2 g^2 + 2^-80 D^2) |w_v|^2 / 3), and the result's to
    u / sqrt(3) of it (f16: or 2^-25 / sqrt(3) each); twice that is allowed.  A logit is off by (width / 16 + 1) 2^-22
    of its terms' sizes, lse by that and 2^-20 and half a step (2^-20 below 32): p by their sum."""
    from bafe_b200 import lm
    vocab, width, top = 50000, 256, 2.0 ** 14
    u = torch.finfo(dtype).eps / 2
    x = torch.randn(rows, width, generator=gen(1), device="cuda").to(dtype)
    w = (torch.randn(vocab, width, generator=gen(2), device="cuda") / 8).to(dtype)
    target = torch.randint(0, vocab, (rows,), generator=gen(3), device="cuda")
    dloss = top * 2.0 ** -(torch.arange(rows, device="cuda") % 25).float()
    _, lse = lm.linear_cross_entropy(x, w, target)
    dx, _ = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    x64, w64 = x.double(), w.double()
    z = x64 @ w64.t()
    assert float(torch.logsumexp(z, -1).max()) < 32
    zerr = (width / 16 + 1) * 2.0 ** -22 * (x64.abs() @ w64.abs().t()).amax(-1)
    p = torch.softmax(z, -1)
    perr = (p * (2 * zerr + 2.0 ** -19)[:, None]) * dloss.double()[:, None]
    g = p.clone()
    g[torch.arange(rows), target] -= 1.0
    g *= dloss.double()[:, None]
    want = g @ w64
    least, tiny = (2.0 ** -40 * top, 2.0 ** -25 * width ** 0.5) if dtype == torch.float16 else (0.0, 0.0)
    each = torch.sqrt((u * u * g.square() + least * least) @ w64.square().sum(-1) / 3)
    bound = 2 * (each + (u * want.norm(dim=-1) + tiny) / 3 ** 0.5) + (perr @ w64.abs()).norm(dim=-1)
    off = (dx.double() - want).norm(dim=-1)
    assert (off <= bound).all(), float((off / bound).max())


def drift(got, want):
    """Mean relative error, its sign kept: a rounding's is 0."""
    return float(((got.double() - want) / want).mean())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sums_over_very_many_rows_do_not_drift(cuda, dtype):
    """dw over 2^22 rows of one sign.  The tensor core truncates its 32-bit sum at every step of 16 rows, which makes it
    short by some 2^-23 of itself.  Parts of 4096 rows (f16; bf16: 16384) are 256 (1024) steps: short by 2^-15 (2^-13) at
    most, a sixteenth of the type's half step u (a thirty-second); they are added up rounded to nearest, on
    average by nothing.  g's and the results' roundings cancel in the mean over 32 x 64 results, up to 4 times u /
    sqrt(2048)."""
    from bafe_b200 import lm
    rows, vocab, width = 1 << 22, 48, 64
    u = torch.finfo(dtype).eps / 2
    x = (1.0 + torch.rand(rows, width, generator=gen(4), device="cuda")).to(dtype)
    w = (torch.randn(vocab, width, generator=gen(5), device="cuda") / 32).to(dtype)
    target = 32 + torch.randint(0, 16, (rows,), generator=gen(6), device="cuda")      # words 0 .. 31: g = p > 0
    dloss = 2.0 ** -10 * (1.0 + torch.rand(rows, generator=gen(7), device="cuda"))
    _, lse = lm.linear_cross_entropy(x, w, target)
    _, dw = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    want = torch.zeros(32, width, dtype=torch.float64, device="cuda")
    for a in range(0, rows, 1 << 18):
        s = slice(a, a + (1 << 18))
        p = torch.softmax(x[s].double() @ w.double().t(), -1)[:, :32] * dloss[s, None].double()
        want += p.t() @ x[s].double()
    assert abs(drift(dw[:32], want)) < u / 16 + 4 * u / 2048 ** 0.5


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sums_over_very_many_words_do_not_drift(cuda, rows, dtype):
    """dx over 2^22 words of one sign but the target's, whose weights are 0: in splits and pieces, each in parts as above."""
    from bafe_b200 import lm
    vocab, width = 1 << 22, 64
    u = torch.finfo(dtype).eps / 2
    w = torch.rand(vocab, width, generator=gen(8), device="cuda").add_(1.0).to(dtype)
    x = (torch.randn(rows, width, generator=gen(9), device="cuda") / 32).to(dtype)
    target = torch.randint(0, vocab, (rows,), generator=gen(10), device="cuda")
    w[target] = 0
    dloss = torch.ones(rows, device="cuda")
    _, lse = lm.linear_cross_entropy(x, w, target)
    dx, _ = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)
    parts = [torch.logsumexp(x.double() @ w[a:a + (1 << 18)].double().t(), -1) for a in range(0, vocab, 1 << 18)]
    lse64 = torch.logsumexp(torch.stack(parts), 0)[:, None]
    want = torch.zeros(rows, width, dtype=torch.float64, device="cuda")
    for a in range(0, vocab, 1 << 18):
        part = w[a:a + (1 << 18)].double()
        want += torch.exp(x.double() @ part.t() - lse64) @ part
    count = rows * width
    assert abs(drift(dx, want)) < u / 16 + 2.0 ** -17 + 4 * u / count ** 0.5
