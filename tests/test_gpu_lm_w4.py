"""matvec_w4 against the formula in 64 bits.

Tolerances.  Each 128 consecutive x of a row are rounded to 2^-22 of the
largest of them at most (e4m3 not at all); the normal and uniform rows here
keep that below 2^-16 of the sum of magnitudes of 128.  Products and sums
over 128 are exact; what rounds besides are the joining of the bytes' sums,
the scales' products and the sums over groups, warps and slices, each below
2^-22 of the sum of magnitudes for every step.  A chain has at most k / 32 + 64
steps here, below 2^7 for the k of these tests: 2^-14 of the sum of
magnitudes covers them all.
The stored result is off by at most half a step more.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

SUMS = 2.0 ** -14


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def problem(m, n, k, group, xtype, stype, zeros, seed=1, pad=0, shift=0):
    g = gen(seed)
    groups = -(-k // group)
    x = torch.randn(m, k, generator=g, device="cuda")
    xs = None
    if xtype == torch.float8_e4m3fn:
        xs = x.abs().amax(-1) / 448.0
        x = (x / xs[:, None]).to(xtype)
    else:
        x = x.to(xtype)
    qb = (k + 1) // 2
    buf = torch.randint(0, 256, (n * (qb + pad) + 32,), generator=g, device="cuda", dtype=torch.uint8)
    q = buf[shift:shift + n * (qb + pad)].view(n, qb + pad)[:, :qb]
    s = (0.01 + 0.02 * torch.rand(n, groups, generator=g, device="cuda")).to(stype)
    z = torch.randint(0, 16, (n, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return x, xs, q, s, z


def formula(x, xs, q, s, z, group):
    k = x.shape[1]
    at = torch.arange(k, device="cuda")
    v = ((q[:, at // 2].to(torch.int32) >> (4 * (at % 2)).to(torch.int32)) & 15).double()
    zz = z[:, at // group].double() if z is not None else 8.0
    w = (v - zz) * s[:, at // group].double()
    xd = x.double() * (xs.double()[:, None] if xs is not None else 1.0)
    return xd @ w.t(), xd.abs() @ w.abs().t()


def close(y, want, mags):
    tol = torch.finfo(y.dtype).eps / 2 * want.abs() + SUMS * mags + torch.finfo(y.dtype).smallest_normal
    err = (y.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst by {float((err - tol).max())}"


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float8_e4m3fn, torch.bfloat16),
         (torch.bfloat16, torch.float32), (torch.float8_e4m3fn, torch.float32)]
SIZES = [  # rows, n, k, group
    (1, 16, 128, 128), (1, 1, 1, 32), (3, 5, 31, 32), (2, 17, 33, 32), (1, 4096, 4096, 128), (7, 33, 255, 64),
    (8, 64, 1000, 64), (9, 100, 2200, 64), (16, 48, 640, 32), (17, 1531, 777, 96), (32, 80, 8192, 128),
    (5, 40, 8192, 256), (2, 3000, 300, 4096), (33, 30, 500, 32), (70, 20, 4100, 128), (31, 2500, 1024, 64),
]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("xtype,stype", TYPES)
@pytest.mark.parametrize("m,n,k,group", SIZES)
def test_product(cuda, m, n, k, group, xtype, stype, zeros):
    from bafe_b200 import lm
    x, xs, q, s, z = problem(m, n, k, group, xtype, stype, zeros, seed=m + n + k)
    y = lm.matvec_w4(x, q, s, z, group=group, x_scale=xs)
    want, mags = formula(x, xs, q, s, z, group)
    assert y.dtype == (xtype if xs is None else torch.bfloat16)
    close(y, want, mags)


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 2), (4, 4), (8, 8), (16, 0), (16, 16)])
@pytest.mark.parametrize("k,group", [(512, 128), (512, 64), (512, 32), (500, 128), (129, 32)])
def test_weight_alignments(cuda, k, group, pad, shift):
    """Rows that start and end off the wide loads' boundaries."""
    from bafe_b200 import lm
    x, xs, q, s, z = problem(3, 50, k, group, torch.bfloat16, torch.bfloat16, True, seed=9, pad=pad, shift=shift)
    close(lm.matvec_w4(x, q, s, z, group=group), *formula(x, xs, q, s, z, group))


def test_strides_and_out(cuda):
    from bafe_b200 import lm
    x, _, q, s, z = problem(4, 70, 384, 128, torch.float16, torch.float16, True, seed=3)
    big = torch.zeros(4, 500, device="cuda", dtype=torch.float16)
    big[:, 1:385] = x
    s2 = torch.zeros(70, 9, device="cuda", dtype=torch.float16)
    s2[:, 2:5] = s
    z2 = torch.full((70, 9), 7, device="cuda", dtype=torch.uint8)
    z2[:, 2:5] = z
    out = torch.full((4, 100), 3.0, device="cuda", dtype=torch.float16)
    got = lm.matvec_w4(big[:, 1:385], q, s2[:, 2:5], z2[:, 2:5], out=out[:, 5:75])
    close(got, *formula(x, None, q, s, z, 128))
    assert (out[:, :5] == 3).all() and (out[:, 75:] == 3).all()
    assert torch.equal(got, lm.matvec_w4(x, q, s, z))


def test_same_bits_for_a_row_alone(cuda):
    """A row's result does not depend on the rows beside it while the launch is cut alike."""
    from bafe_b200 import lm
    x, _, q, s, z = problem(8, 300, 1024, 128, torch.bfloat16, torch.bfloat16, True, seed=4)
    y = lm.matvec_w4(x, q, s, z)
    for i in range(8):
        assert torch.equal(lm.matvec_w4(x[i:i + 1], q, s, z)[0], y[i])
    assert torch.equal(lm.matvec_w4(x, q, s, z), y)


def test_infinities_and_nan(cuda):
    """They reach the outputs of their own row and no other."""
    from bafe_b200 import lm
    x, _, q, s, z = problem(4, 64, 200, 64, torch.bfloat16, torch.bfloat16, False, seed=5)
    clean = lm.matvec_w4(x, q, s, z, group=64)
    x = x.clone()
    x[1, 3] = float("nan")
    x[2, 199] = float("inf")
    y = lm.matvec_w4(x, q, s, z, group=64)
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
    # scales of infinity mark their own column
    s = s.clone()
    s[7, 0] = float("inf")
    y = lm.matvec_w4(x[:1], q, s, z, group=64)
    assert not torch.isfinite(y[0, 7]) and torch.equal(y[0, :7], clean[0, :7])


def test_no_rows_no_outputs(cuda):
    from bafe_b200 import lm
    x, _, q, s, z = problem(4, 64, 200, 64, torch.bfloat16, torch.bfloat16, False)
    assert lm.matvec_w4(x[:0], q, s, group=64).shape == (0, 64)
    assert lm.matvec_w4(x, q[:0], s[:0], group=64).shape == (4, 0)


def test_stream_and_graphs(cuda):
    """k cut into slices (few outputs, long k) uses scratch: two graphs in turn, and another stream."""
    from bafe_b200 import lm
    a = problem(6, 32, 8192, 128, torch.bfloat16, torch.bfloat16, True, seed=6)
    b = problem(6, 32, 8192, 128, torch.bfloat16, torch.bfloat16, True, seed=7)
    run = lambda p, **kw: lm.matvec_w4(p[0], p[2], p[3], p[4], **kw)   # noqa: E731
    want = [run(p) for p in (a, b)]
    close(want[0], *formula(*a, 128))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = run(a, stream=side)
    side.synchronize()
    assert torch.equal(got, want[0])
    graphs = []
    for p in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = run(p)
        graphs.append((g, r))
    for _ in range(3):
        graphs[0][0].replay()
        graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want[0]) and torch.equal(graphs[1][1], want[1])


def test_refusals(cuda):
    from bafe_b200 import lm
    x, _, q, s, z = problem(4, 64, 256, 64, torch.bfloat16, torch.bfloat16, True)
    bad = [lambda: lm.matvec_w4(x, q, s, z, group=48), lambda: lm.matvec_w4(x, q, s, z, group=128),
           lambda: lm.matvec_w4(x, q[:, :-1], s, z, group=64), lambda: lm.matvec_w4(x, q, s, z[:-1], group=64),
           lambda: lm.matvec_w4(x, q.cpu(), s, z, group=64), lambda: lm.matvec_w4(x.to(torch.float8_e4m3fn), q, s, z, group=64),
           lambda: lm.matvec_w4(x, q, s, z, group=64, x_scale=torch.ones(4, device="cuda")),
           lambda: lm.matvec_w4(x, q, s, z, group=64, out=torch.empty(4, 64, device="cuda", dtype=torch.float16)),
           lambda: lm.matvec_w4(x.t().contiguous().t(), q, s, z, group=64)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call in (lambda: lm.matvec_w4(x.float(), q, s, z, group=64), lambda: lm.matvec_w4(x, q, s.double(), z, group=64),
                 lambda: lm.matvec_w4(x, q, s, z.int(), group=64)):
        with pytest.raises(TypeError):
            call()
