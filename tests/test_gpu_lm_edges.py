"""Calls of the language-model operators that their documentation allows and
that are easily forgotten: mixed types, one buffer for input and output,
extreme values, the same tensor twice, sizes that change from call to call.
Tolerances as in the operators' own test files."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def near(got, want, rel, floor=0.0):
    err = (got.double() - want).abs()
    bad = ~(err <= rel * want.abs() + floor)
    assert not bad.any(), f"{int(bad.sum())} outside, worst {float(err.max())}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [512, 515, 17000])
def test_norm_gradient_with_f32_weight(cuda, dtype, width):
    from bafe_b200 import lm
    h, dy, w = randn((40, width), dtype, 1), randn((40, width), dtype, 2), randn((width,), torch.float32, 3)
    dx, dw = lm.rms_norm_grad(dy, h, w)
    assert dx.dtype == dtype and dw.dtype == torch.float32
    hd, g = h.double(), dy.double() * w.double()
    r = 1.0 / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-6)
    parts = (r * g).abs() + (hd * r ** 3).abs() * (g * hd).abs().mean(-1, keepdim=True)
    near(dx, r * g - hd * r ** 3 * (g * hd).mean(-1, keepdim=True), torch.finfo(dtype).eps / 2 + 2.0 ** -17,
         2.0 ** -17 * parts + torch.finfo(dtype).smallest_normal)
    terms = dy.double() * hd * r
    near(dw, terms.sum(0), 2.0 ** -24, 512 * 2.0 ** -24 * terms.abs().sum(0))


def test_columns_of_one_buffer(cuda):
    """Input and output side by side in the same rows; neither disturbs the other."""
    from bafe_b200 import lm
    buf = randn((30, 640), torch.bfloat16, 4)
    keep = buf.clone()
    w = randn((256,), torch.bfloat16, 5)
    x, out = buf[:, :256], buf[:, 320:576]
    want = lm.rms_norm(x.contiguous(), w)
    assert torch.equal(lm.rms_norm(x, w, out=out), want)
    assert torch.equal(buf[:, :320], keep[:, :320]) and torch.equal(buf[:, 576:], keep[:, 576:])
    buf.copy_(keep)
    we, off = randn((2, 200, 256), torch.bfloat16, 6, 0.1), torch.tensor([0, 11, 30], dtype=torch.int32, device="cuda")
    want = lm.grouped_matmul(x.contiguous(), we, off)
    assert torch.equal(lm.grouped_matmul(x, we, off, out=buf[:, 300:500]), want)
    assert torch.equal(buf[:, :300], keep[:, :300]) and torch.equal(buf[:, 500:], keep[:, 500:])
    with pytest.raises(ValueError):
        lm.rms_norm(x, w, out=buf[:, 200:456])
    one = buf[:1, :256]
    with pytest.raises(ValueError):       # the same place in another type
        lm.rms_norm_e4m3(one, w, out=one.view(torch.float8_e4m3fn)[:, :256])


def test_same_tensor_twice(cuda):
    from bafe_b200 import lm
    x, w = randn((20, 384), torch.float16, 7), randn((384,), torch.float16, 8)
    y, h = lm.rms_norm(x, w, x)
    assert torch.equal(h, x + x) and torch.equal(y, lm.rms_norm(x + x, w))
    x2 = x.clone()
    y2, h2 = lm.rms_norm(x2, w, x2, residual_out=x2)
    assert h2 is x2 and torch.equal(h2, h) and torch.equal(y2, y)
    off = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    dw = lm.grouped_matmul_grad_weight(x, x, off)
    want = x.double().t() @ x.double()
    near(dw[0], want, 2.0 ** -11, 2.0 ** -14 * (x.double().abs().t() @ x.double().abs()))


def test_w4_extreme_rows(cuda):
    """Rows near the ends of the range, a row with one value far above the others, a row of zeros."""
    from bafe_b200 import lm
    k, n = 640, 96
    q = torch.randint(0, 256, (n, k // 2), generator=gen(9), device="cuda", dtype=torch.uint8)
    s = 0.5 + torch.rand(n, k // 128, generator=gen(10), device="cuda")
    x = randn((6, k), torch.bfloat16, 11)
    x[0] *= 1e-30
    x[1] *= 1e30
    x[2, 77] = 1000.0
    x[3] = 0
    x[4] = x[4].abs()                         # all of one sign: zero points and sums cancel
    y = lm.matvec_w4(x, q, s)
    at = torch.arange(k, device="cuda")
    w = (((q[:, at // 2].int() >> (4 * (at % 2)).int()) & 15).double() - 8) * s[:, at // 128].double()
    want, mags = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    near(y, want, 2.0 ** -8, 2.0 ** -14 * mags)
    assert (y[3] == 0).all()
    big = x.clone()
    big[5, 600] = float("-inf")
    y2 = lm.matvec_w4(big, q, s)
    assert torch.equal(y2[:5], y[:5]) and torch.isnan(y2[5]).all()


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 16, 17, 32, 33, 64])
def test_w4_row_counts(cuda, rows):
    from bafe_b200 import lm
    k, n, group = 1152, 200, 128
    q = torch.randint(0, 256, (n, k // 2), generator=gen(12), device="cuda", dtype=torch.uint8)
    s, z = 0.1 + torch.rand(n, 9, generator=gen(13), device="cuda").half(), torch.randint(0, 16, (n, 9), generator=gen(14), device="cuda", dtype=torch.uint8)
    x = randn((rows, k), torch.float16, 15)
    at = torch.arange(k, device="cuda")
    w = (((q[:, at // 2].int() >> (4 * (at % 2)).int()) & 15).double() - z[:, at // group].double()) * s[:, at // group].double()
    near(lm.matvec_w4(x, q, s, z, group=group), x.double() @ w.t(), 2.0 ** -11, 2.0 ** -14 * (x.double().abs() @ w.abs().t()))


def test_sizes_that_change_from_call_to_call(cuda):
    """What one call's checks found does not answer for another's."""
    from bafe_b200 import lm
    w = randn((256,), torch.bfloat16, 16)
    for rows in (3, 1, 300, 3):
        x = randn((rows, 256), torch.bfloat16, rows)
        assert lm.rms_norm(x, w).shape == (rows, 256)
    with pytest.raises(TypeError):
        lm.rms_norm(x.double(), w)
    with pytest.raises(ValueError):
        lm.rms_norm(x, w.cpu())
    with pytest.raises(ValueError):
        lm.rms_norm(x, w, x.t().contiguous().t())
    with pytest.raises(ValueError):
        lm.rms_norm(x, w, residual_out=x)
    off = torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda")
    we = randn((2, 64, 256), torch.bfloat16, 17)
    lm.grouped_matmul(x, we, off)
    with pytest.raises(ValueError):
        lm.grouped_matmul_grad_input(x, we, off)
    with pytest.raises(ValueError):
        lm.grouped_matmul(x, we, off[:2])
    q = torch.randint(0, 256, (64, 128), generator=gen(18), device="cuda", dtype=torch.uint8)
    s = torch.ones(64, 2, device="cuda")
    lm.matvec_w4(x, q, s, group=128)
    with pytest.raises(ValueError):
        lm.matvec_w4(x, q, s, group=64)
    assert lm.matvec_w4(x, q, torch.ones(64, 1, device="cuda"), group=256).shape == (3, 64)


@pytest.mark.parametrize("first,last", [(0, 0), (5, 5), (0, 64), (64, 64), (63, 64)])
def test_group_borders(cuda, first, last):
    """Groups that start and end anywhere, among empty ones; the rest of the output untouched."""
    from bafe_b200 import lm
    x, w = randn((64, 96), torch.bfloat16, 19), randn((4, 72, 96), torch.bfloat16, 20, 0.1)
    off = torch.tensor([first, first, last, last, last], dtype=torch.int32, device="cuda")
    out = torch.full((64, 72), 2.0, device="cuda", dtype=torch.bfloat16)
    y = lm.grouped_matmul(x, w, off, out=out)
    assert (y[:first] == 2).all() and (y[last:] == 2).all()
    want = x[first:last].double() @ w[1].double().t()
    near(y[first:last], want, 2.0 ** -8, 2.0 ** -14 * (x[first:last].double().abs() @ w[1].double().abs().t()))
    dw = lm.grouped_matmul_grad_weight(out, x, off)
    assert all((dw[e] == 0).all() for e in (0, 2, 3))
    want = out[first:last].double().t() @ x[first:last].double()
    near(dw[1], want, 2.0 ** -8, 2.0 ** -14 * (out[first:last].double().abs().t() @ x[first:last].double().abs()))


def test_every_remainder_of_a_group(cuda):
    """Experts of 0 to 70 rows one after the other: every way a contraction ends inside a block of 64."""
    from bafe_b200 import lm
    sizes = list(range(71))
    rows = sum(sizes)
    off = torch.tensor(list(itertools.accumulate([0] + sizes)), dtype=torch.int32, device="cuda")
    x, dy = randn((rows, 40), torch.float16, 21), randn((rows, 24), torch.float16, 22)
    dw = lm.grouped_matmul_grad_weight(dy, x, off)
    w = randn((71, 24, 40), torch.float16, 23)
    y, dx = lm.grouped_matmul(x, w, off), lm.grouped_matmul_grad_input(dy, w, off)
    at = 0
    for e, z in enumerate(sizes):
        a, b = dy[at:at + z].double(), x[at:at + z].double()
        near(dw[e], a.t() @ b, 2.0 ** -11, 2.0 ** -14 * (a.abs().t() @ b.abs()) + 1e-7)
        near(y[at:at + z], b @ w[e].double().t(), 2.0 ** -11, 2.0 ** -14 * (b.abs() @ w[e].double().abs().t()) + 1e-7)
        near(dx[at:at + z], a @ w[e].double(), 2.0 ** -11, 2.0 ** -14 * (a.abs() @ w[e].double().abs()) + 1e-7)
        at += z


@pytest.mark.parametrize("rows", [1, 2, 5, 16, 32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_weights_at_their_zero_point(cuda, rows, group):
    """Channels whose weights all equal their zero points give exact zeros,
    and so do columns that only such weights meet."""
    from bafe_b200 import lm
    k, n = 1280, 75
    z = torch.randint(0, 16, (n, k // group), generator=gen(24), device="cuda", dtype=torch.uint8)
    q = z.repeat_interleave(group // 2, 1) * 17
    s = 0.5 + torch.rand(n, k // group, generator=gen(25), device="cuda")
    x = randn((rows, k), torch.bfloat16, 26).abs() * 1000
    assert (lm.matvec_w4(x, q, s, z, group=group) == 0).all()
    half = (z[::3] ^ 8).repeat_interleave(group // 2, 1) * 17       # every third channel 8 away everywhere
    q[::3] = half
    y = lm.matvec_w4(x, q, s, z, group=group)
    w = ((half & 15).double() - z[::3].repeat_interleave(group // 2, 1).double()).repeat_interleave(2, 1)
    w *= s[::3].double().repeat_interleave(group, 1)
    near(y[:, ::3], x.double() @ w.t(), 2.0 ** -8, 2.0 ** -14 * (x.double().abs() @ w.abs().t()))
    assert (y[:, 1::3] == 0).all() and (y[:, 2::3] == 0).all()
    assert (lm.matvec_w4(x, torch.full_like(q, 0x88), s, group=group) == 0).all()      # without zero points: 8


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [512, 515, 17000])
@pytest.mark.parametrize("power", [-50, 50])
def test_norm_gradient_of_very_small_and_large_rows(cuda, dtype, width, power):
    """r^3 is out of 32-bit range here, dx is not."""
    from bafe_b200 import lm
    h, dy, w = randn((9, width), dtype, 27, 2.0 ** power), randn((9, width), dtype, 28), randn((width,), dtype, 29)
    dx, dw = lm.rms_norm_grad(dy, h, w, eps=0.0)
    hd, g = h.double(), dy.double() * w.double()
    r = 1.0 / torch.sqrt(hd.square().mean(-1, keepdim=True))
    parts = (r * g).abs() + (hd * r ** 3).abs() * (g * hd).abs().mean(-1, keepdim=True)
    near(dx, r * g - hd * r ** 3 * (g * hd).mean(-1, keepdim=True), torch.finfo(dtype).eps / 2 + 2.0 ** -17,
         2.0 ** -17 * parts)
    terms = dy.double() * hd * r
    near(dw, terms.sum(0), torch.finfo(dtype).eps / 2, 512 * 2.0 ** -24 * terms.abs().sum(0))


def test_refuses_arguments_of_other_kinds(cuda):
    from bafe_b200 import lm
    x, w = randn((4, 128), torch.bfloat16, 30), randn((128,), torch.bfloat16, 31)
    lm.rms_norm(x, w)                                    # the checks of what follows find these known
    for eps in (-1.0, float("nan")):
        with pytest.raises(RuntimeError, match="eps"):
            lm.rms_norm(x, w, eps=eps)
        with pytest.raises(RuntimeError, match="eps"):
            lm.rms_norm_grad(x, x, w, eps=eps)
    for call in (lambda: lm.rms_norm(x, w, eps="small"),
                 lambda: lm.rms_norm(x, w, out=[0.0]), lambda: lm.rms_norm(x, w, stream=0),
                 lambda: lm.rms_norm(x, w, out=x.cpu()), lambda: lm.rms_norm(x, w, x, residual_out="h"),
                 lambda: lm.rms_norm_grad(x, x, w, weight_out=3),
                 lambda: lm.rms_norm_e4m3(x, w, scale_out=x.view(-1)[:8].view(torch.float32))):
        with pytest.raises((TypeError, ValueError)):
            call()
    q, s = torch.zeros(16, 64, device="cuda", dtype=torch.uint8), torch.ones(16, 1, device="cuda")
    lm.matvec_w4(x, q, s, group=128)
    off, we = torch.tensor([0, 4], dtype=torch.int32, device="cuda"), randn((1, 16, 128), torch.bfloat16, 32)
    x8, s8 = lm.rms_norm_e4m3(x, w)
    for call in (lambda: lm.matvec_w4(x, q, s, group=128.0), lambda: lm.matvec_w4(x, q, s, group=None),
                 lambda: lm.matvec_w4(x, q, s, out=0), lambda: lm.matvec_w4(x8, q, s, x_scale=s8, out=0),
                 lambda: lm.grouped_matmul(x, we, off, out=0), lambda: lm.grouped_matmul(x, we, off, stream="s"),
                 lambda: lm.grouped_matmul_grad_weight(x, x, off, out=())):
        with pytest.raises((TypeError, ValueError)):
            call()
    import numpy as np
    assert torch.equal(lm.rms_norm(x, w, eps=np.float32(0.5)), lm.rms_norm(x, w, eps=0.5))
    assert torch.equal(lm.matvec_w4(x, q, s, group=np.int64(128)), lm.matvec_w4(x, q, s))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("k,base", [(77, 0), (78, 2), (80, 1), (333, 3)])
@pytest.mark.parametrize("marks", [[0, 5, 5, 9, 40], [3, 3, 20, 20, 33], [0, 30, 12, 35, 35], [-4, 7, 50, 2, 40]])
def test_rows_off_16_byte_boundaries(cuda, dtype, k, base, marks):
    """Operands that are copied first give what the same values on boundaries
    give, whichever experts have rows (also by offsets out of order)."""
    from bafe_b200 import lm
    n, rows = 50, 40
    x, w = randn((rows, k), torch.float32, 33).to(dtype), randn((4, n, k), torch.float32, 34).to(dtype)
    es = x.element_size()
    xa, wa = torch.zeros(rows, 384, device="cuda", dtype=dtype)[:, :k], torch.zeros(4, n, 384, device="cuda", dtype=dtype)[..., :k]
    xu = torch.zeros(rows * k + 8, device="cuda", dtype=dtype)[base:base + rows * k].view(rows, k)
    wu = torch.zeros(4 * n * k + 8, device="cuda", dtype=dtype)[base:base + 4 * n * k].view(4, n, k)
    for to, of in ((xa, x), (xu, x), (wa, w), (wu, w)):
        to.view(torch.uint8 if es == 1 else torch.int16).copy_(of.view(torch.uint8 if es == 1 else torch.int16))
    off = torch.tensor(marks, device="cuda", dtype=torch.int32)
    scales = {}
    if es == 1:
        scales = {"x_scale": 0.5 + torch.rand(rows, generator=gen(35), device="cuda"),
                  "w_scale": 0.5 + torch.rand(4, n, generator=gen(36), device="cuda")}
    out = lambda: torch.full((rows, n), 3.0, device="cuda", dtype=torch.bfloat16 if es == 1 else dtype)
    want = lm.grouped_matmul(xa, wa, off, out=out(), **scales)
    assert torch.equal(lm.grouped_matmul(xu, wu, off, out=out(), **scales), want)
    top, e = 0, []
    for m in marks:
        top = max(top, min(max(m, 0), rows))
        e.append(top)
    s = scales.get("x_scale", torch.ones(rows, device="cuda")).double()
    c = scales.get("w_scale", torch.ones(4, n, device="cuda")).double()
    for i in range(4):
        a, b = x[e[i]:e[i + 1]].double() * s[e[i]:e[i + 1], None], w[i].double() * c[i][:, None]
        near(want[e[i]:e[i + 1]], a @ b.t(), torch.finfo(want.dtype).eps / 2, 2.0 ** -14 * (a.abs() @ b.abs().t()) + 1e-7)
    assert (want[:e[0]] == 3).all() and (want[e[4]:] == 3).all()


@pytest.mark.parametrize("n,k", [(70, 66), (33, 130), (40, 7), (300, 258)])
@pytest.mark.parametrize("pad", [0, 1, 2, 6])
def test_results_off_16_byte_boundaries(cuda, n, k, pad):
    """Result rows that start anywhere; what lies between them stays."""
    from bafe_b200 import lm
    x, dy = randn((90, k), torch.bfloat16, 37), randn((90, n), torch.bfloat16, 38)
    off = torch.tensor([0, 37, 37, 90], device="cuda", dtype=torch.int32)
    buf = torch.full((3, n, k + pad), 5.0, device="cuda", dtype=torch.bfloat16)
    dw = lm.grouped_matmul_grad_weight(dy, x, off, out=buf[..., :k])
    assert (buf[..., k:] == 5).all() and (dw[1] == 0).all()
    for e, (a, b) in ((0, (0, 37)), (2, (37, 90))):
        p, q = dy[a:b].double(), x[a:b].double()
        near(dw[e], p.t() @ q, 2.0 ** -8, 2.0 ** -14 * (p.abs().t() @ q.abs()) + 1e-7)
    w = randn((3, n, k), torch.bfloat16, 39)
    rows = torch.full((90, n + pad), 5.0, device="cuda", dtype=torch.bfloat16)
    y = lm.grouped_matmul(x, w, off, out=rows[:, :n])
    assert (rows[:, n:] == 5).all()
    for e, (a, b) in ((0, (0, 37)), (2, (37, 90))):
        q, v = x[a:b].double(), w[e].double()
        near(y[a:b], q @ v.t(), 2.0 ** -8, 2.0 ** -14 * (q.abs() @ v.abs().t()) + 1e-7)


@pytest.mark.parametrize("rows", [16, 17, 31, 40])
def test_w4_many_weights_in_several_launches(cuda, rows):
    from bafe_b200 import lm
    k, n = 8192, 8200
    q = torch.randint(0, 256, (n, k // 2), generator=gen(40), device="cuda", dtype=torch.uint8)
    s = 0.1 + torch.rand(n, k // 128, generator=gen(41), device="cuda").bfloat16()
    x = randn((rows, k), torch.bfloat16, 42)
    w = torch.stack((q & 15, q >> 4), -1).reshape(n, k).double() - 8
    w *= s.double().repeat_interleave(128, 1)
    near(lm.matvec_w4(x, q, s), x.double() @ w.t(), 2.0 ** -8, 2.0 ** -14 * (x.double().abs() @ w.abs().t()))
