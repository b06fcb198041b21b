"""Products grouped by expert, and their gradients, against 64-bit sums.

Tolerances.  Products of 16-bit (or e4m3) values are exact in 32 bits.  The
tensor core adds 16 (32) of them and its accumulator per step, dropping bits
below the largest term: at most 2^-22 of the sum of magnitudes a step, and
at most 4096 / 16 steps here: 2^-14.  The e4m3 scales add two products
(2^-23).  The stored result is off by at most half a step more.
"""
import itertools
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

SUMS = 2.0 ** -14
ROOT = Path(__file__).resolve().parent.parent


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def offsets_of(sizes, first=0):
    return torch.tensor(list(itertools.accumulate([first] + list(sizes))), dtype=torch.int32, device="cuda")


def close(y, want, mags, name=""):
    tol = torch.finfo(y.dtype).eps / 2 * want.abs() + SUMS * mags + torch.finfo(y.dtype).smallest_normal
    err = (y.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} outside, first {bad.nonzero()[:4].tolist()}"


def check_forward(y, x, w, sizes, first=0, xs=None, ws=None):
    at = first
    for e, z in enumerate(sizes):
        a, b = x[at:at + z].double(), w[e].double()
        if xs is not None:
            a, b = a * xs[at:at + z, None].double(), b * ws[e][:, None].double()
        close(y[at:at + z], a @ b.t(), a.abs() @ b.abs().t(), f"expert {e}")
        at += z


SIZES = [  # rows of each expert, n, k
    ([1], 64, 64), ([5], 256, 128), ([256], 256, 64), ([257, 3], 512, 192), ([0, 7, 0, 0, 33, 1, 0], 300, 136),
    ([64, 64, 64, 64], 1024, 512), ([700, 0, 90, 513], 264, 1000), ([31, 32, 33, 95, 96, 97, 127, 128, 129], 320, 264),
    ([1] * 40, 128, 4096), ([0, 0, 3000], 520, 72), ([0] * 63 + [2], 2048, 256), ([255, 256, 1], 8, 8),
    ([2, 40], 33, 51), ([70, 300], 257, 1001), ([9], 1, 1), ([3, 0, 2], 4096, 40),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,n,k", SIZES)
def test_forward(cuda, sizes, n, k, dtype):
    import bafe_b200
    from bafe_b200 import lm
    x, w = randn((sum(sizes), k), dtype, 1), randn((len(sizes), n, k), dtype, 2, 0.1)
    y = lm.grouped_matmul(x, w, offsets_of(sizes))
    bafe_b200.synchronize()
    assert y.dtype == dtype and y.shape == (sum(sizes), n)
    check_forward(y, x, w, sizes)


@pytest.mark.parametrize("out", [None, torch.float16])
@pytest.mark.parametrize("sizes,n,k", SIZES)
def test_forward_e4m3(cuda, sizes, n, k, out):
    import bafe_b200
    from bafe_b200 import lm
    rows, e = sum(sizes), len(sizes)
    x, w = randn((rows, k), torch.float32, 3, 50.0).to(torch.float8_e4m3fn), randn((e, n, k), torch.float32, 4, 50.0).to(torch.float8_e4m3fn)
    xs = 0.01 * (0.5 + torch.rand(rows, generator=gen(5), device="cuda"))
    ws = 0.01 * (0.5 + torch.rand(e, n, generator=gen(6), device="cuda"))
    o = None if out is None else torch.zeros(rows, n, device="cuda", dtype=out)
    y = lm.grouped_matmul(x, w, offsets_of(sizes), x_scale=xs, w_scale=ws, out=o)
    bafe_b200.synchronize()
    assert y.dtype == (out or torch.bfloat16)
    check_forward(y, x, w, sizes, xs=xs, ws=ws)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,n,k", SIZES)
def test_grad_input(cuda, sizes, n, k, dtype):
    import bafe_b200
    from bafe_b200 import lm
    dy, w = randn((sum(sizes), n), dtype, 7), randn((len(sizes), n, k), dtype, 8, 0.1)
    dx = lm.grouped_matmul_grad_input(dy, w, offsets_of(sizes))
    bafe_b200.synchronize()
    check_forward(dx, dy, w.transpose(1, 2), sizes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,n,k", SIZES)
def test_grad_weight(cuda, sizes, n, k, dtype):
    import bafe_b200
    from bafe_b200 import lm
    dy, x = randn((sum(sizes), n), dtype, 9), randn((sum(sizes), k), dtype, 10)
    dw = lm.grouped_matmul_grad_weight(dy, x, offsets_of(sizes))
    bafe_b200.synchronize()
    at = 0
    for e, z in enumerate(sizes):
        a, b = dy[at:at + z].double().t(), x[at:at + z].double()
        close(dw[e], a @ b, a.abs() @ b.abs(), f"expert {e}")
        at += z


def test_gradients_against_differences(cuda):
    """Central differences of sum(y * c) in 64 bits at a few places."""
    from bafe_b200 import lm
    sizes, n, k = [3, 0, 70], 24, 40
    off = offsets_of(sizes)
    x, w, c = randn((73, k), torch.float16, 11), randn((3, n, k), torch.float16, 12), randn((73, n), torch.float16, 13)
    dx = lm.grouped_matmul_grad_input(c, w, off)
    dw = lm.grouped_matmul_grad_weight(c, x, off)
    owner = torch.tensor([0] * 3 + [2] * 70, device="cuda")

    def loss(x, w):
        return (torch.einsum("tk,tnk->tn", x, w[owner]) * c.double()).sum()
    h = 1e-3
    for t, i in ((0, 0), (2, 39), (50, 17)):
        e = torch.zeros(73, k, device="cuda", dtype=torch.float64)
        e[t, i] = h
        num = float(loss(x.double() + e, w.double()) - loss(x.double() - e, w.double())) / (2 * h)
        assert abs(num - float(dx[t, i])) <= 2e-3 * max(1.0, abs(num))
    for ex, j, i in ((0, 0, 0), (2, 23, 39), (1, 4, 4)):
        e = torch.zeros(3, n, k, device="cuda", dtype=torch.float64)
        e[ex, j, i] = h
        num = float(loss(x.double(), w.double() + e) - loss(x.double(), w.double() - e)) / (2 * h)
        assert abs(num - float(dw[ex, j, i])) <= 2e-3 * max(1.0, abs(num))


def test_rows_outside_the_groups(cuda):
    """Rows before the first and behind the last group are neither written nor read into a sum, whatever they hold."""
    from bafe_b200 import lm
    sizes, first, n, k = [20, 0, 45], 5, 136, 72
    x, w, dy = randn((90, k), torch.bfloat16, 14), randn((3, n, k), torch.bfloat16, 15), randn((90, n), torch.bfloat16, 16)
    for t in (x, dy):
        t[:5] = float("nan")
        t[70:] = float("inf")
    off = offsets_of(sizes, first)
    out = torch.full((90, n), 7.0, device="cuda", dtype=torch.bfloat16)
    y = lm.grouped_matmul(x, w, off, out=out)
    assert y is out and (y[:5] == 7).all() and (y[70:] == 7).all()
    check_forward(y, x, w, sizes, first)
    dw = lm.grouped_matmul_grad_weight(dy, x, off)
    at = first
    for e, z in enumerate(sizes):
        a, b = dy[at:at + z].double().t(), x[at:at + z].double()
        close(dw[e], a @ b, a.abs() @ b.abs(), f"expert {e}")
        at += z


def test_nan_stays_with_its_expert(cuda):
    from bafe_b200 import lm
    for sizes in ([10, 10, 10], [64, 3, 61], [1, 1, 1], [130, 200, 70]):
        n, k, off = 96, 80, offsets_of(sizes)
        rows = sum(sizes)
        x, dy = randn((rows, k), torch.float16, 17), randn((rows, n), torch.float16, 18)
        w = randn((3, n, k), torch.float16, 19)
        clean_y, clean_dw = lm.grouped_matmul(x, w, off), lm.grouped_matmul_grad_weight(dy, x, off)
        a, b = sizes[0], sizes[0] + sizes[1]
        x2, dy2 = x.clone(), dy.clone()
        x2[a:b], dy2[a:b] = float("nan"), float("inf")
        y, dw = lm.grouped_matmul(x2, w, off), lm.grouped_matmul_grad_weight(dy2, x2, off)
        assert torch.equal(y[:a], clean_y[:a]) and torch.equal(y[b:], clean_y[b:]) and torch.isnan(y[a:b]).all()
        assert torch.equal(dw[0], clean_dw[0]) and torch.equal(dw[2], clean_dw[2]) and torch.isnan(dw[1]).all()


def test_strides_and_storage_orders(cuda):
    """Padded rows, weights stored with either dimension contiguous, unaligned starts."""
    from bafe_b200 import lm
    sizes, n, k = [40, 0, 21], 100, 88
    off = offsets_of(sizes)
    x, w, dy = randn((61, k), torch.bfloat16, 20), randn((3, n, k), torch.bfloat16, 21), randn((61, n), torch.bfloat16, 22)
    want, want_dx = lm.grouped_matmul(x, w, off), lm.grouped_matmul_grad_input(dy, w, off)
    want_dw = lm.grouped_matmul_grad_weight(dy, x, off)
    check_forward(want, x, w, sizes)
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(lm.grouped_matmul(x, wt, off), want)
    assert torch.equal(lm.grouped_matmul_grad_input(dy, wt, off), want_dx)
    for shift in (1, 8):
        xb = torch.zeros(61, 120, device="cuda", dtype=torch.bfloat16)
        xb[:, shift:shift + k] = x
        wb = torch.zeros(3, 104, 96, device="cuda", dtype=torch.bfloat16)
        wb[:, :n, shift:shift + k] = w
        dyb = torch.zeros(61, 120, device="cuda", dtype=torch.bfloat16)
        dyb[:, shift:shift + n] = dy
        xv, wv, dyv = xb[:, shift:shift + k], wb[:, :n, shift:shift + k], dyb[:, shift:shift + n]
        assert torch.equal(lm.grouped_matmul(xv, wv, off), want)
        assert torch.equal(lm.grouped_matmul_grad_input(dyv, wv, off), want_dx)
        out = torch.full((3, n + 3, k + 5), 9.0, device="cuda", dtype=torch.bfloat16)
        got = lm.grouped_matmul_grad_weight(dyv, xv, off, out=out[:, :n, 2:2 + k])
        assert torch.equal(got, want_dw)
        assert (out[:, n:] == 9).all() and (out[:, :, :2] == 9).all() and (out[:, :, 2 + k:] == 9).all()
        out = torch.full((61, n + 7), 9.0, device="cuda", dtype=torch.bfloat16)
        assert torch.equal(lm.grouped_matmul(x, w, off, out=out[:, 3:3 + n]), want)
        assert (out[:, :3] == 9).all() and (out[:, 3 + n:] == 9).all()


def test_offsets_are_clamped(cuda):
    """Offsets outside the rows or out of order address nothing else."""
    from bafe_b200 import lm
    x, w = randn((50, 64), torch.bfloat16, 23), randn((4, 32, 64), torch.bfloat16, 24)
    out = torch.full((50, 32), 5.0, device="cuda", dtype=torch.bfloat16)
    bad = torch.tensor([-7, 20, 10, 30, 1 << 30], dtype=torch.int32, device="cuda")
    y = lm.grouped_matmul(x, w, bad, out=out)
    check_forward(y, x, w, [20, 0, 10, 20])
    dw = lm.grouped_matmul_grad_weight(y, x, bad)
    assert (dw[1] == 0).all() and torch.isfinite(dw).all()


def test_most_experts(cuda):
    from bafe_b200 import lm
    sizes = [(i * 7) % 5 for i in range(1024)]
    x, w = randn((sum(sizes), 64), torch.bfloat16, 25), randn((1024, 16, 64), torch.bfloat16, 26)
    off = offsets_of(sizes)
    y = lm.grouped_matmul(x, w, off)
    owner = torch.repeat_interleave(torch.arange(1024, device="cuda"), torch.tensor(sizes, device="cuda"))
    want = torch.einsum("tk,tnk->tn", x.double(), w[owner].double())
    mags = torch.einsum("tk,tnk->tn", x.double().abs(), w[owner].double().abs())
    close(y, want, mags)
    dw = lm.grouped_matmul_grad_weight(y, x, off)
    assert (dw[0] == 0).all() and (dw[5] == 0).all()
    close(dw[1], y[:2].double().t() @ x[:2].double(), y[:2].double().abs().t() @ x[:2].double().abs())


def test_no_rows(cuda):
    from bafe_b200 import lm
    w, off = randn((3, 32, 64), torch.bfloat16, 27), offsets_of([0, 0, 0])
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    assert lm.grouped_matmul(x, w, off).shape == (0, 32)
    dw = lm.grouped_matmul_grad_weight(x[:, :32], x, off, out=torch.ones(3, 32, 64, device="cuda", dtype=torch.bfloat16))
    assert (dw == 0).all()


def test_same_bits_every_run(cuda):
    from bafe_b200 import lm
    sizes, n, k = [300, 17, 0, 515], 520, 264
    off = offsets_of(sizes)
    x, w, dy = randn((832, k), torch.bfloat16, 28), randn((4, n, k), torch.bfloat16, 29), randn((832, n), torch.bfloat16, 30)
    first = None
    for _ in range(5):
        got = (lm.grouped_matmul(x, w, off), lm.grouped_matmul_grad_input(dy, w, off), lm.grouped_matmul_grad_weight(dy, x, off))
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(got, first))
        first = got


def test_streams_and_graphs(cuda):
    """Unaligned operands use scratch: two graphs in turn, and another stream beside the current one."""
    from bafe_b200 import lm
    sizes, n, k = [30, 0, 101], 77, 51
    off = offsets_of(sizes)
    xs = [randn((131, k), torch.bfloat16, 31 + i) for i in range(2)]
    w = randn((3, n, k), torch.bfloat16, 33)
    want = [lm.grouped_matmul(x, w, off) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = [lm.grouped_matmul(xs[0], w, off, stream=side), lm.grouped_matmul(xs[1], w, off)]
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = lm.grouped_matmul(x, w, off)
        graphs.append((g, r))
    off2 = offsets_of([100, 31, 0])
    want2 = [lm.grouped_matmul(x, w, off2) for x in xs]
    for _ in range(3):
        for g, _r in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want[0]) and torch.equal(graphs[1][1], want[1])
    off.copy_(off2)                     # other group sizes in the captured call
    for g, _r in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want2[0]) and torch.equal(graphs[1][1], want2[1])


def test_first_call_inside_a_capture(cuda):
    """A process whose first call of each operator is captured."""
    code = """
import sys; sys.path.insert(0, sys.argv[1])
import torch
from bafe_b200 import lm
x = torch.randn(64, 128, device="cuda").bfloat16(); w = torch.randn(2, 64, 128, device="cuda").bfloat16()
off = torch.tensor([0, 10, 64], dtype=torch.int32, device="cuda"); g1 = torch.ones(128, device="cuda").bfloat16()
q = torch.randint(0, 256, (64, 64), device="cuda", dtype=torch.uint8); s = torch.ones(64, 1, device="cuda").bfloat16()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    n = lm.rms_norm(x, g1); y = lm.grouped_matmul(n, w, off); dw = lm.grouped_matmul_grad_weight(y, n, off)
    dx = lm.grouped_matmul_grad_input(y, w, off); d, dg = lm.rms_norm_grad(dx, x, g1); v = lm.matvec_w4(x[:3], q, s)
g.replay(); torch.cuda.synchronize()
got = [t.clone() for t in (n, y, dw, dx, d, dg, v)]
n = lm.rms_norm(x, g1); y = lm.grouped_matmul(n, w, off); dw = lm.grouped_matmul_grad_weight(y, n, off)
dx = lm.grouped_matmul_grad_input(y, w, off); d, dg = lm.rms_norm_grad(dx, x, g1); v = lm.matvec_w4(x[:3], q, s)
assert all(torch.equal(a, b) for a, b in zip(got, (n, y, dw, dx, d, dg, v)))
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code, str(ROOT / "bafe-basic-algibra-fusion-engine-_b200")],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_refusals(cuda):
    from bafe_b200 import lm
    x, w, off = randn((8, 64), torch.bfloat16, 34), randn((2, 32, 64), torch.bfloat16, 35), offsets_of([3, 5])
    x8, w8 = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    xs, ws = torch.ones(8, device="cuda"), torch.ones(2, 32, device="cuda")
    bad = [lambda: lm.grouped_matmul(x[:, :32], w, off), lambda: lm.grouped_matmul(x, w[0], off),
           lambda: lm.grouped_matmul(x, w, off.long()), lambda: lm.grouped_matmul(x, w, off[:2]),
           lambda: lm.grouped_matmul(x, w, off.cpu()), lambda: lm.grouped_matmul(x, w, off, x_scale=xs),
           lambda: lm.grouped_matmul(x8, w8, off), lambda: lm.grouped_matmul(x8, w8, off, x_scale=xs, w_scale=ws[:1]),
           lambda: lm.grouped_matmul(x8, w8.transpose(1, 2).contiguous().transpose(1, 2), off, x_scale=xs, w_scale=ws),
           lambda: lm.grouped_matmul(x, w[:1].expand(2, 32, 64), off), lambda: lm.grouped_matmul(x, w[:, ::2, ::2], off),
           lambda: lm.grouped_matmul(x, w, off, out=x[:, :32]),
           lambda: lm.grouped_matmul_grad_input(x[:, :32], w.cpu(), off),
           lambda: lm.grouped_matmul_grad_weight(x[:4], x, off), lambda: lm.grouped_matmul_grad_weight(x, x.half(), off),
           lambda: lm.grouped_matmul_grad_weight(x, x, off, out=torch.empty(2, 64, 32, device="cuda", dtype=x.dtype))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call in (lambda: lm.grouped_matmul(x.float(), w, off), lambda: lm.grouped_matmul(x, w.half(), off),
                 lambda: lm.grouped_matmul_grad_input(x8[:, :32], w8, off)):
        with pytest.raises(TypeError):
            call()
