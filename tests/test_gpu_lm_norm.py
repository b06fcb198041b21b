"""rms_norm, its e4m3 form and its gradient against plain formulas in 64 bits.

Tolerances.  A stored result is rounded once: half a step, eps / 2 of its
type, relative to the value.  Before that the kernels compute in 32 bits:
the sum of squares is a chain of at most 128 additions a thread (rows up to
2^17) and 10 levels of pairs, so its relative error is below 138 * 2^-24,
half of that in r; rsqrtf (2 ulp), the mean, eps and three products add
fewer than 16 * 2^-24.  F32 = 2^-17 covers them.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -17
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def formula(x, w, res, eps):
    h = x if res is None else (x.double() + res.double()).to(x.dtype)
    # one rounding of the exact sum: the 32-bit sum of two 16-bit values is
    # exact or rounds the same way but for double rounding at a tie
    hd = h.double()
    r = 1.0 / torch.sqrt(hd.square().mean(-1, keepdim=True) + eps)
    return h, hd * r * w.double(), r


def near(got, want, rel, floor=None, name=""):
    err = (got.double() - want).abs()
    tol = rel * want.abs()
    if floor is not None:
        tol = tol + floor
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} outside, worst {float((err - tol).max())}"


SHAPES = [(1, 1), (3, 7), (5, 32), (2, 33), (9, 64), (1, 4096), (13, 4096), (3, 5003), (300, 72), (2000, 16),
          (2, 8192), (1, 16384), (2, 32768), (2, 32776), (3, 70001), (1, 131072), (400, 1024)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
def test_norm(cuda, rows, width, dtype):
    from bafe_b200 import lm
    x, w = make((rows, width), dtype, 1), make((width,), dtype, 2)
    y = lm.rms_norm(x, w, eps=1e-5)
    _, want, _ = formula(x, w, None, 1e-5)
    assert y.dtype == dtype
    near(y, want, half_step(dtype) + F32, floor=torch.finfo(dtype).smallest_normal, name="y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
def test_norm_residual_and_e4m3(cuda, rows, width, dtype):
    from bafe_b200 import lm
    x, res = make((rows, width), dtype, 3), make((rows, width), dtype, 4, 3.0)
    w = make((width,), torch.float32, 5)
    y, h = lm.rms_norm(x, w, res)
    q, s, h8 = lm.rms_norm_e4m3(x, w, res)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32 and s.shape == (rows,)
    # the stored sum: at most half a step (and the 32-bit sum's) off the exact one
    exact = x.double() + res.double()
    near(h, exact, torch.finfo(dtype).eps / 2 + 2.0 ** -24, name="h")
    assert torch.equal(h, h8)
    r = 1.0 / torch.sqrt(h.double().square().mean(-1, keepdim=True) + 1e-6)
    want = h.double() * r * w.double()
    near(y, want, half_step(dtype) + F32, floor=torch.finfo(dtype).smallest_normal, name="y")
    top = want.abs().amax(-1)
    near(s, top / 448.0, F32, name="scale")
    # e4m3: half a step is 2^-4 of a normal value, 2^-10 below the normals
    near(q.double() * s.double()[:, None], want, 2.0 ** -4 + F32, floor=2.0 ** -10 * s.double()[:, None] * (1 + F32),
         name="q")


def test_rows_that_leave_nothing(cuda):
    """Zero rows, rows of the smallest and largest values, NaN and infinity."""
    from bafe_b200 import lm
    for dtype in TYPES:
        w = torch.ones(64, device="cuda", dtype=dtype)
        x = torch.zeros(6, 64, device="cuda", dtype=dtype)
        x[1, 3] = torch.finfo(dtype).smallest_normal
        x[2] = 2.0 ** 15
        x[3, 5] = float("nan")
        x[4, 6] = float("inf")
        x[5] = -1.0
        y = lm.rms_norm(x, w).float()
        q, s = lm.rms_norm_e4m3(x, w)
        v = q.float() * s[:, None]
        assert (y[0] == 0).all() and (v[0] == 0).all() and s[0] == 1
        assert torch.isfinite(y[1]).all() and torch.isfinite(v[1]).all() and torch.isfinite(s[1])
        assert torch.allclose(y[2], torch.ones_like(y[2]), rtol=2e-2) and torch.allclose(v[2], y[2], rtol=0.07)
        assert torch.isnan(y[3]).all() and torch.isnan(v[3]).all() and s[3] == 1
        assert torch.isnan(y[4, 6]) and (y[4, :6] == 0).all() and torch.isnan(v[4, 6])
        assert torch.allclose(y[5], torch.full_like(y[5], -1.0), rtol=2e-2)
        near(v[5], y[5].double(), 2.0 ** -4 + 2.0 ** -8, name="last")
        # a weight of NaN marks the row's 8-bit values, whatever the row's sum
        w2 = w.clone()
        w2[1] = float("nan")
        q2, s2 = lm.rms_norm_e4m3(x, w2)
        assert torch.isnan(q2.float()[5, 1]) and s2[5] == 1


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_offsets_and_in_place(cuda, dtype):
    """Padded rows, rows that start off a 16-byte boundary, outputs over inputs."""
    from bafe_b200 import lm
    big = make((7, 300), dtype, 6)
    w = make((257,), dtype, 7)[1:]
    for x in (big[:, :256], big[:, 1:257], big[:, 8:264]):
        want = formula(x, w, None, 1e-6)[1]
        near(lm.rms_norm(x, w), want, half_step(dtype) + F32, floor=torch.finfo(dtype).smallest_normal)
        out = torch.full((7, 400), 9.0, device="cuda", dtype=dtype)
        got = lm.rms_norm(x, w, out=out[:, 3:259])
        near(got, want, half_step(dtype) + F32, floor=torch.finfo(dtype).smallest_normal)
        assert (out[:, :3] == 9).all() and (out[:, 259:] == 9).all()
    for width in (256, 250, 40000):
        x, res, w = make((4, width), dtype, 8), make((4, width), dtype, 9), make((width,), dtype, 10)
        y0, h0 = lm.rms_norm(x, w, res)
        x1, r1 = x.clone(), res.clone()
        y1, h1 = lm.rms_norm(x1, w, r1, out=x1, residual_out=r1)
        assert y1 is x1 and h1 is r1 and torch.equal(y0, y1) and torch.equal(h0, h1)
        x2 = x.clone()
        assert torch.equal(lm.rms_norm(x2, w, out=x2), lm.rms_norm(x, w))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_dh", [False, True])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (2, 33), (1, 4096), (700, 4096), (5, 5003), (3000, 16),
                                        (65, 8192), (3, 16384), (3, 32776), (2, 70001), (1500, 72)])
def test_gradient_formula(cuda, rows, width, dtype, with_dh):
    from bafe_b200 import lm
    h, dy = make((rows, width), dtype, 11), make((rows, width), dtype, 12, 0.1)
    w = make((width,), dtype, 13)
    dh = make((rows, width), dtype, 14, 0.1) if with_dh else None
    dx, dw = lm.rms_norm_grad(dy, h, w, dh)
    hd, dyd, wd = h.double(), dy.double(), w.double()
    r = 1.0 / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-6)
    g = dyd * wd
    back = hd * r ** 3 * (g * hd).mean(-1, keepdim=True)
    want = r * g - back + (dh.double() if with_dh else 0.0)
    # the terms cancel: their 32-bit errors are relative to each of them,
    # the mean's to the mean of the magnitudes
    parts = (r * g).abs() + (hd * r ** 3).abs() * (g * hd).abs().mean(-1, keepdim=True)
    near(dx, want, half_step(dtype) + F32, floor=F32 * parts + torch.finfo(dtype).smallest_normal, name="dx")
    terms = dyd * hd * r
    # a slot adds rows / slots terms, a column 8 chains of slots / 8: fewer
    # than 512 additions here
    near(dw, terms.sum(0), half_step(dtype) + 2.0 ** -24, floor=512 * 2.0 ** -24 * terms.abs().sum(0) +
         torch.finfo(dtype).smallest_normal, name="dw")


def test_gradient_against_differences(cuda):
    """Central differences of sum(y * c) + sum(h * d) in 64 bits."""
    from bafe_b200 import lm
    x, w = make((3, 24), torch.float32, 15), make((24,), torch.float32, 16)
    c, d = make((3, 24), torch.float32, 17).double(), make((3, 24), torch.float32, 18).double()

    def loss(x, w):
        r = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        return ((x * r * w) * c).sum() + (x * d).sum()
    dx, dw = lm.rms_norm_grad(c.float(), x, w, d.float())
    step = 1e-5
    for i, j in ((0, 0), (1, 13), (2, 23)):
        e = torch.zeros(3, 24, device="cuda", dtype=torch.float64)
        e[i, j] = step
        num = (loss(x.double() + e, w.double()) - loss(x.double() - e, w.double())) / (2 * step)
        assert abs(float(num) - float(dx[i, j])) < 1e-4 * max(1.0, abs(float(num)))
        num = (loss(x.double(), w.double() + e[i]) - loss(x.double(), w.double() - e[i])) / (2 * step)
        assert abs(float(num) - float(dw[j])) < 1e-4 * max(1.0, abs(float(num)))


def test_gradient_in_place_and_repeatable(cuda):
    from bafe_b200 import lm
    for width in (512, 511, 40000):
        h, dy, w = make((50, width), torch.bfloat16, 19), make((50, width), torch.bfloat16, 20), make((width,), torch.bfloat16, 21)
        dh = make((50, width), torch.bfloat16, 22)
        a = lm.rms_norm_grad(dy, h, w, dh)
        b = lm.rms_norm_grad(dy, h, w, dh)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        for which in ("dy", "dh"):
            dy2, dh2 = dy.clone(), dh.clone()
            got = lm.rms_norm_grad(dy2, h, w, dh2, out=dy2 if which == "dy" else dh2)
            assert torch.equal(got[0], a[0]) and torch.equal(got[1], a[1])


def test_no_rows(cuda):
    from bafe_b200 import lm
    x, w = make((0, 64), torch.bfloat16, 1), make((64,), torch.bfloat16, 2)
    assert lm.rms_norm(x, w).shape == (0, 64)
    q, s = lm.rms_norm_e4m3(x, w)
    assert q.shape == (0, 64) and s.shape == (0,)
    dx, dw = lm.rms_norm_grad(x, x, w)
    assert dx.shape == (0, 64) and (dw == 0).all()


def test_other_stream_and_graph(cuda):
    """On a stream of the caller's, and captured: two graphs, replayed in turn, keep scratch of their own."""
    from bafe_b200 import lm
    h, dy, w = make((300, 1024), torch.bfloat16, 23), make((300, 1024), torch.bfloat16, 24), make((1024,), torch.bfloat16, 25)
    h2 = make((300, 1024), torch.bfloat16, 26)
    want, want2 = lm.rms_norm_grad(dy, h, w), lm.rms_norm_grad(dy, h2, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = lm.rms_norm_grad(dy, h, w, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for v in (h, h2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = lm.rms_norm_grad(dy, v, w)
        graphs.append((g, r))
    for _ in range(3):
        graphs[0][0].replay()
        graphs[1][0].replay()
    torch.cuda.synchronize()
    for (g, r), t in zip(graphs, (want, want2)):
        assert torch.equal(r[0], t[0]) and torch.equal(r[1], t[1])


def test_launch_count(cuda):
    import bafe_b200
    from bafe_b200 import lm
    x, w = make((4, 64), torch.bfloat16, 1), make((64,), torch.bfloat16, 2)
    n = bafe_b200.launch_count()
    lm.rms_norm(x, w)
    lm.rms_norm_grad(x, x, w)
    assert bafe_b200.launch_count() - n == 3


def test_refusals(cuda):
    from bafe_b200 import lm
    x, w = make((4, 64), torch.bfloat16, 1), make((64,), torch.bfloat16, 2)
    with pytest.raises(ValueError):
        lm.rms_norm(x, w[:32])
    with pytest.raises(TypeError):
        lm.rms_norm(x, w.half())
    with pytest.raises(TypeError):
        lm.rms_norm(x.double(), w)
    with pytest.raises(ValueError):
        lm.rms_norm(x, w, x[:2])
    with pytest.raises(ValueError):
        lm.rms_norm(x, w, x.half())
    with pytest.raises(ValueError):
        lm.rms_norm(x.t(), w)
    with pytest.raises(ValueError):
        lm.rms_norm(x, w, x.cpu())
    with pytest.raises(ValueError):
        lm.rms_norm(x, w, residual_out=torch.empty_like(x))
    with pytest.raises(ValueError):
        lm.rms_norm(x, w, out=torch.empty(4, 63, device="cuda", dtype=x.dtype))
    with pytest.raises(ValueError):
        lm.rms_norm(x[:1].expand(4, 64), w)
    with pytest.raises(RuntimeError):
        lm.rms_norm(x, w, eps=-1.0)
    with pytest.raises(RuntimeError):
        lm.rms_norm(x, w, eps=float("nan"))
    out = torch.empty(5, 64, device="cuda", dtype=x.dtype)
    with pytest.raises(ValueError):       # y over the stored sum
        lm.rms_norm(x, w, x, out=out[:4], residual_out=out[:4])
    with pytest.raises(ValueError):       # y over x, a row later
        lm.rms_norm(out[:4], w, out=out[1:])
