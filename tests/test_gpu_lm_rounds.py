"""Grouped products of more tiles than pairs of SMs, with contractions of many
blocks and of every length: ragged ends land on other stages of the ring from
round to round, and the two accumulators alternate.  Every expert's result is
compared with 64-bit sums; tolerances as in test_gpu_lm_grouped.py (at most
4096 / 16 steps of 2^-22 of the sum of magnitudes, the e4m3 scales 2^-23, and
half a step of the stored type)."""
import itertools
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

SUMS = 2.0 ** -14


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def offsets_of(sizes, first=0):
    return torch.tensor(list(itertools.accumulate([first] + list(sizes))), dtype=torch.int32, device="cuda")


def close(y, want, mags, name):
    tol = torch.finfo(y.dtype).eps / 2 * want.abs() + SUMS * mags + torch.finfo(y.dtype).smallest_normal
    bad = ~((y.double() - want).abs() <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} outside, first {bad.nonzero()[:4].tolist()}"


def ragged(experts, top, seed):
    rng = random.Random(seed)
    return [0 if rng.random() < 0.1 else rng.randint(1, top) for _ in range(experts)]


CASES = [  # experts, most rows of one, n, k
    (40, 300, 520, 264), (90, 300, 264, 520), (130, 129, 256, 256), (37, 1000, 777, 130), (300, 70, 128, 513),
    (20, 300, 1024, 1000),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts,top,n,k", CASES)
def test_weight_gradient(cuda, experts, top, n, k, dtype):
    import bafe_b200
    from bafe_b200 import lm
    sizes = ragged(experts, top, experts)
    rows = sum(sizes)
    dy, x = randn((rows + 9, n), dtype, 1), randn((rows + 9, k), dtype, 2)
    dy[:4], x[:4], dy[rows + 4:], x[rows + 4:] = (float("nan"),) * 4
    dw = lm.grouped_matmul_grad_weight(dy, x, offsets_of(sizes, 4))
    bafe_b200.synchronize()
    at = 4
    for e, z in enumerate(sizes):
        a, b = dy[at:at + z].double().t(), x[at:at + z].double()
        close(dw[e], a @ b, a.abs() @ b.abs(), f"expert {e} of {z} rows")
        at += z
    assert torch.equal(lm.grouped_matmul_grad_weight(dy, x, offsets_of(sizes, 4)), dw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("experts,top,n,k", CASES)
def test_forward_and_rows_gradient(cuda, experts, top, n, k, dtype):
    import bafe_b200
    from bafe_b200 import lm
    sizes = ragged(experts, top, experts + 1)
    rows, off, to8 = sum(sizes), offsets_of(sizes), dtype == torch.float8_e4m3fn
    x, w = randn((rows, k), torch.float32, 3).to(dtype), randn((experts, n, k), torch.float32, 4).to(dtype)
    scales = {}
    if to8:
        scales = {"x_scale": 0.01 * (0.5 + torch.rand(rows, generator=gen(5), device="cuda")),
                  "w_scale": 0.5 + torch.rand(experts, n, generator=gen(6), device="cuda")}
    y = lm.grouped_matmul(x, w, off, **scales)
    dy = randn((rows, n), torch.float32, 7).to(torch.bfloat16 if to8 else dtype)
    dx = None if to8 else lm.grouped_matmul_grad_input(dy, w, off)
    bafe_b200.synchronize()
    at = 0
    for e, z in enumerate(sizes):
        a, b = x[at:at + z].double(), w[e].double()
        if to8:
            a, b = a * scales["x_scale"][at:at + z, None].double(), b * scales["w_scale"][e][:, None].double()
        close(y[at:at + z], a @ b.t(), a.abs() @ b.abs().t(), f"expert {e} of {z} rows")
        if dx is not None:
            a = dy[at:at + z].double()
            close(dx[at:at + z], a @ b, a.abs() @ b.abs(), f"gradient, expert {e} of {z} rows")
        at += z


@pytest.mark.parametrize("rows", [33, 128, 129, 400])
def test_few_rows_over_many_tiles(cuda, rows):
    """The rings for few rows over several rounds, and the call just above them."""
    from bafe_b200 import lm
    experts, n, k = 24, 1100, 1000
    rng = random.Random(rows)
    marks = sorted(rng.randint(0, rows) for _ in range(experts - 1))
    sizes = [b - a for a, b in zip([0] + marks, marks + [rows])]
    x, w = randn((rows, k), torch.bfloat16, 8), randn((experts, n, k), torch.bfloat16, 9)
    y = lm.grouped_matmul(x, w, offsets_of(sizes))
    dx = lm.grouped_matmul_grad_input(y, w, offsets_of(sizes))
    at = 0
    for e, z in enumerate(sizes):
        a, b = x[at:at + z].double(), w[e].double()
        close(y[at:at + z], a @ b.t(), a.abs() @ b.abs().t(), f"expert {e}")
        a = y[at:at + z].double()
        close(dx[at:at + z], a @ b, a.abs() @ b.abs(), f"gradient, expert {e}")
        at += z
