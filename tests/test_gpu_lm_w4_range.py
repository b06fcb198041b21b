"""matvec_w4 on tokens whose values differ widely in size.

Tolerance as in test_gpu_lm_w4.py: 2^-14 of the sum of |x w| of the output's
own terms and half a step of the stored type.  Products of a token's 16-bit
value and an integer weight of up to 8 bits are exact in 32 bits; an
instruction adds 16 of them to its 32-bit sum (at most 2^-22 of their
magnitudes), 8 instructions a scale unit, and then one multiply-add per
unit, warp and slice (2^-24 each, fewer than 2^9 of them here): below 2^-14
together.  Terms that are zero (a weight at its zero point) count for nothing
in that sum, however large their token is.  Results below the normal range
are off by a step of the subnormals at most: half of one in the rounding, far
less in 32 bits' own subnormals before it.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

SUMS = 2.0 ** -14


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weights(n, k, group, seed, top=16):
    """Random weights and zero points below `top`, and scales."""
    q = torch.randint(0, 16, (n, k), generator=gen(seed), device="cuda", dtype=torch.uint8)
    z = torch.randint(0, top, (n, -(-k // group)), generator=gen(seed + 1), device="cuda", dtype=torch.uint8)
    s = 0.01 + 0.02 * torch.rand(n, -(-k // group), generator=gen(seed + 2), device="cuda")
    return q, z, s


def packed(q):
    if q.shape[1] % 2:
        q = torch.cat((q, torch.zeros_like(q[:, :1])), 1)
    return q[:, ::2] | q[:, 1::2] << 4


def check(y, x, q, z, s, group, xs=None):
    at = torch.arange(q.shape[1], device="cuda") // group
    w = (q.double() - z.double()[:, at]) * s.double()[:, at]
    xd = x.double() * (1.0 if xs is None else xs.double()[:, None])
    want, mags = xd @ w.t(), xd.abs() @ w.abs().t()
    tol = torch.finfo(y.dtype).eps / 2 * want.abs() + SUMS * mags + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    err = (y.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst {float((err / (mags + 1e-300)).max())} of the magnitudes"


LARGE = [(torch.bfloat16, 1e4), (torch.bfloat16, 1e5), (torch.bfloat16, 1e6), (torch.bfloat16, 1e12),
         (torch.float16, 1e4), (torch.float16, 6e4)]


@pytest.mark.parametrize("rows", [1, 2, 5, 8, 16, 31])
@pytest.mark.parametrize("group", [32, 64, 128, 96])
@pytest.mark.parametrize("dtype,large", LARGE)
def test_large_values_at_the_zero_point(cuda, dtype, large, group, rows):
    """One value of every 128 far above the rest; in every other output its weight is the zero point."""
    from bafe_b200 import lm
    n, k = 90, 1152
    q, z, s = weights(n, k, group, 1)
    s *= 0.1                                             # f16 results stay in range
    x = torch.randn(rows, k, generator=gen(4), device="cuda") * (1.0 if large < 6e4 else 0.01)
    at = torch.arange(0, k, 128, device="cuda") + torch.randint(0, 128, (k // 128,), generator=gen(5), device="cuda")
    x[:, at] = large
    q[::2, at] = z[::2, at // group]
    x = x.to(dtype)
    check(lm.matvec_w4(x, packed(q), s, z, group=group), x, q, z, s, group)


@pytest.mark.parametrize("rows", [1, 8, 20])
@pytest.mark.parametrize("dtype,large", LARGE[1:])
def test_large_values_in_a_group_of_small_scale(cuda, dtype, large, rows):
    """The group that holds them counts for little in the result."""
    from bafe_b200 import lm
    n, k, group = 70, 1024, 32
    q, z, s = weights(n, k, group, 7)
    s[:, ::4] *= 1e-3 / large
    x = torch.randn(rows, k, generator=gen(8), device="cuda")
    x.view(rows, -1, 4, 32)[:, :, 0] *= large / 8
    x = x.to(dtype)
    check(lm.matvec_w4(x, packed(q), s, z, group=group), x, q, z, s, group)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("rows", [1, 3, 9, 32])
def test_every_magnitude_in_one_row(cuda, dtype, rows):
    """Values spread evenly over the type's exponents, subnormal ones too; each output sees one part of them only."""
    from bafe_b200 import lm
    k, group, parts = 1280, 64, 16
    info = torch.finfo(dtype)
    low, high = (-30.0, 60.0) if dtype == torch.bfloat16 else (-24.0, 15.0) if dtype == torch.float16 else (-9.0, 8.0)
    power = torch.rand(rows, k, generator=gen(9), device="cuda") * (high - low) + low
    sign = torch.randint(0, 2, (rows, k), generator=gen(10), device="cuda") * 2 - 1
    x = (torch.exp2(power) * sign).clamp(-info.max, info.max).to(dtype)
    n = 4 * parts
    q, z, s = weights(n, k, group, 11)
    # output i: weights at the zero point but where the first row's power lies in part i % parts
    part = ((power[0] - low) / (high - low) * parts).int().clamp(0, parts - 1)
    out = torch.arange(n, device="cuda")[:, None] % parts != part[None]
    q = torch.where(out, z[:, torch.arange(k, device="cuda") // group], q)
    xs = None
    if dtype == torch.float8_e4m3fn:
        xs = 0.5 + torch.rand(rows, generator=gen(12), device="cuda")
    s16 = (0.01 * s).to(torch.bfloat16)
    y = lm.matvec_w4(x[:1], packed(q), s16, z, group=group, x_scale=None if xs is None else xs[:1])
    check(y, x[:1], q, z, s16, group, None if xs is None else xs[:1])
    y = lm.matvec_w4(x, packed(q), s16, z, group=group, x_scale=xs)
    check(y, x, q, z, s16, group, xs)


@pytest.mark.parametrize("xtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 4, 12, 24])
def test_zero_points_of_a_whole_byte(cuda, rows, group, xtype):
    """Zero points may be any byte; those of 128 and more stand beside small ones."""
    from bafe_b200 import lm
    n, k = 77, 896
    q, z, s = weights(n, k, group, 13, top=256)
    z[5::7] = 255
    z[6::7] &= 127
    x = torch.randn(rows, k, generator=gen(16), device="cuda").to(xtype)
    xs = 0.5 + torch.rand(rows, generator=gen(17), device="cuda") if xtype == torch.float8_e4m3fn else None
    check(lm.matvec_w4(x, packed(q), s, z, group=group, x_scale=xs), x, q, z, s, group, xs)


@pytest.mark.parametrize("rows", [1, 7, 16, 30])
def test_rows_at_the_ends_of_the_range(cuda, rows):
    """The largest and the smallest bf16 values, whose sums of q x leave 32 bits' range on their own."""
    from bafe_b200 import lm
    n, k, group = 50, 1024, 128
    q, z, s = weights(n, k, group, 18)
    s *= 0.01
    x = torch.randn(rows, k, generator=gen(19), device="cuda").to(torch.bfloat16)
    x[0] = torch.where(x[0] > 0, 1.0, -1.0) * torch.finfo(torch.bfloat16).max * 0.75
    if rows > 2:
        x[1] *= 1e-37
        x[2, 100:140] *= 2.0 ** 120
    check(lm.matvec_w4(x, packed(q), s, z, group=group), x, q, z, s, group)
    # a single large one among ordinary ones, at the zero point in every other output
    x = torch.randn(rows, k, generator=gen(20), device="cuda").to(torch.bfloat16)
    x[:, 300] = torch.finfo(torch.bfloat16).max
    q[::2, 300] = z[::2, 300 // group]
    check(lm.matvec_w4(x, packed(q), s, z, group=group), x, q, z, s, group)


@pytest.mark.parametrize("where", [0, 127, 128, 700, 1023])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_no_number_marks_its_whole_row(cuda, dtype, value, where):
    """Also where its weight is the zero point, and no other row."""
    from bafe_b200 import lm
    q, z, s = weights(40, 1024, 128, 21)
    q[::2, where] = z[::2, where // 128]
    x = torch.randn(9, 1024, generator=gen(22), device="cuda").to(dtype)
    clean = lm.matvec_w4(x, packed(q), s, z)
    x[3, where] = value
    y = lm.matvec_w4(x, packed(q), s, z)
    assert torch.isnan(y[3]).all()
    assert torch.equal(y[:3], clean[:3]) and torch.equal(y[4:], clean[4:])


def test_rows_beside_a_row_leave_its_bits(cuda):
    """The same launch with other neighbours, and in another order, gives a row the same bits."""
    from bafe_b200 import lm
    for rows, n, k, group in ((8, 300, 1024, 128), (16, 128, 8192, 64), (32, 95, 2048, 32)):
        q, z, s = weights(n, k, group, 23)
        x = torch.randn(rows, k, generator=gen(24), device="cuda").to(torch.bfloat16)
        p = packed(q)
        y = lm.matvec_w4(x, p, s, z, group=group)
        order = torch.randperm(rows, generator=gen(25), device="cuda")
        assert torch.equal(lm.matvec_w4(x[order], p, s, z, group=group), y[order])
        other = torch.randn(rows, k, generator=gen(26), device="cuda").to(torch.bfloat16)
        other[rows // 2] = x[rows // 2]
        assert torch.equal(lm.matvec_w4(other, p, s, z, group=group)[rows // 2], y[rows // 2])
        assert torch.equal(lm.matvec_w4(x, p, s, z, group=group), y)
