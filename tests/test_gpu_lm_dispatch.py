"""The rows' way to the experts and back (lm.dispatch, lm.combine,
lm.combine_grad) against plain indexing in 64 bits.

Bounds.  A sum of k products in 32 bits is off by at most (k + 1) half ulps
(2^-24) of the sum of their sizes, a dot product over `width` elements by at
most width of them, whatever the order; a result's rounding by half a step of
its type (f16: at least half of the smallest, 2^-25).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def places(rows, k, n, seed, lost=0.0):
    """[rows, k] different rows of n; some of them none."""
    p = torch.randperm(n, generator=gen(seed), device="cuda")[:rows * k].int().view(rows, k)
    if lost:
        p[torch.rand(rows, k, generator=gen(seed + 1), device="cuda") < lost] = -1
    return p


SHAPES = [(1, 1, 1), (1, 8, 4096), (5, 3, 33), (70, 6, 250), (300, 8, 1024), (9, 31, 2050), (700, 2, 8), (17, 9, 5003)]


@pytest.mark.parametrize("rows,k,width", SHAPES)
@pytest.mark.parametrize("dtype", TYPES + [torch.float8_e4m3fn])
def test_dispatch(cuda, rows, k, width, dtype):
    from bafe_b200 import lm
    x, n = randn((rows, width), 1, dtype), rows * k + 3
    place = places(rows, k, n, 2, 0.1)
    place[0, 0] = n                                      # outside: no place
    scale = randn((rows,), 3)
    old, old_scale = randn((n, width), 4, dtype), randn((n,), 5)
    y, s = lm.dispatch(x, place, scale=scale, out=old.clone(), scale_out=old_scale.clone())
    raw = (lambda t: t.view(torch.uint8)) if dtype == torch.float8_e4m3fn else (lambda t: t)
    want, want_scale = raw(old).clone(), old_scale.clone()
    for t in range(rows):
        for p in place[t].tolist():
            if 0 <= p < n:
                want[p] = raw(x)[t]
                want_scale[p] = scale[t]
    assert torch.equal(raw(y), want) and torch.equal(s, want_scale)
    full = places(rows, k, rows * k, 6)
    z = lm.dispatch(x, full)
    assert z.shape == (rows * k, width)
    assert torch.equal(raw(z)[full.reshape(-1).long()], raw(x).repeat_interleave(k, 0))


@pytest.mark.parametrize("rows,k,width", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weighted", [True, False])
def test_combine(cuda, rows, k, width, dtype, weighted):
    from bafe_b200 import lm
    n = rows * k + 2
    y, place = randn((n, width), 1, dtype), places(rows, k, n, 2, 0.2)
    place[0] = -1                                        # a row without any
    w = randn((rows, k), 3) if weighted else None
    unused = torch.ones(n, dtype=torch.bool, device="cuda")
    unused[place[place >= 0].long()] = False
    y[unused] = float("nan")                             # rows that no place names do not matter
    got = lm.combine(y, place, w)
    terms = y.double()[place.long().clamp_min(0)] * (place >= 0)[..., None]
    terms = torch.where((place >= 0)[..., None], terms, 0.0) * (1.0 if w is None else w.double()[..., None])
    want, size = terms.sum(1), terms.abs().sum(1)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    bound = (k + 1) * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * (want.abs() + size * 2.0 ** -18) + tiny
    assert ((got.double() - want).abs() <= bound).all()
    assert (got[0] == 0).all()


@pytest.mark.parametrize("rows,k,width", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_combine_grad(cuda, rows, k, width, dtype):
    from bafe_b200 import lm
    n = rows * k + 2
    y, place, w = randn((n, width), 1, dtype), places(rows, k, n, 2, 0.2), randn((rows, k), 3)
    dout = randn((rows, width), 4, dtype)
    old = randn((n, width), 5, dtype)
    dy, dw = lm.combine_grad(dout, y, place, w, out=old.clone())
    some = place >= 0
    terms = torch.where(some[..., None], y.double()[place.long().clamp_min(0)], 0.0) * dout.double()[:, None]
    assert ((dw.double() - terms.sum(-1)).abs() <= width * 2.0 ** -24 * terms.abs().sum(-1) + 1e-38).all()
    want = old.double()
    full = w.double()[..., None] * dout.double()[:, None]
    want[place[some].long()] = full[some]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    named = torch.zeros(n, dtype=torch.bool, device="cuda")
    named[place[some].long()] = True
    bound = (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * want.abs() + tiny
    assert ((dy.double() - want).abs() <= bound)[named].all()
    assert torch.equal(dy[~named], old[~named])
    # in place of y
    held = y.clone()
    dy2, dw2 = lm.combine_grad(dout, held, place, w, out=held)
    assert dy2 is held and torch.equal(dw2, dw) and torch.equal(dy2[named], dy[named]) and torch.equal(dy2[~named], y[~named])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,ld", [(0, 72), (1, 75), (2, 74), (8, 80), (0, 66)])
def test_strides_and_offsets(cuda, dtype, offset, ld):
    """Columns of wider buffers, on and off the boundaries of vectors."""
    from bafe_b200 import lm
    rows, k, width = 40, 4, 64

    def inside(n, seed):
        return torch.as_strided(randn((n * ld + offset,), seed, dtype), (n, width), (ld, 1), offset)

    n = rows * k
    x, y, place, w = inside(rows, 1), inside(n, 2), places(rows, k, n, 3), randn((rows, k + 2), 4)[:, 1:k + 1]
    wide = torch.full((rows, k + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + k] = place
    place2 = wide[:, 2:2 + k]
    out = inside(n, 5)
    assert torch.equal(lm.dispatch(x, place2, out=out), lm.dispatch(x.contiguous(), place))
    assert torch.equal(lm.combine(y, place2, w, out=inside(rows, 6)), lm.combine(y.contiguous(), place, w.contiguous()))
    dy, dw = lm.combine_grad(x, y, place2, w, out=inside(n, 7))
    dy2, dw2 = lm.combine_grad(x.contiguous(), y.contiguous(), place, w.contiguous())
    assert torch.equal(dy, dy2) and torch.allclose(dw, dw2, rtol=0, atol=width * 2.0 ** -23 * 16)
    # one row of gradients and one of weights for all rows
    one, same = x[:1].expand(rows, width), w[:1].expand(rows, k)
    dy3, _ = lm.combine_grad(one, y, place, same)
    dy4, _ = lm.combine_grad(one.contiguous(), y, place, same.contiguous())
    assert torch.equal(dy3, dy4)


def test_rows_beyond_32_bit_offsets(cuda):
    """Rows of y more than 2^31 elements (and 2^32 bytes) from its start."""
    from bafe_b200 import lm
    width, n = 4096, (1 << 19) + 300                     # 2.1e9 elements of 2 bytes
    y = torch.empty(n, width, dtype=torch.bfloat16, device="cuda")
    place = torch.tensor([[n - 1, 5], [7, n - 2]], dtype=torch.int32, device="cuda")
    x = randn((2, width), 1, torch.bfloat16)
    w = torch.tensor([[1.0, 2.0], [0.5, 4.0]], device="cuda")
    lm.dispatch(x, place, out=y)
    assert torch.equal(y[n - 1], x[0]) and torch.equal(y[n - 2], x[1]) and torch.equal(y[7], x[1])
    assert torch.equal(lm.combine(y, place, w).double(), (x.double() * torch.tensor([[3.0], [4.5]], device="cuda")).bfloat16().double())
    dy, _ = lm.combine_grad(x, y, place, w, out=y)
    assert torch.equal(dy[n - 2], x[1] * 4) and torch.equal(dy[5], x[0] * 2)


def test_empty_calls(cuda):
    from bafe_b200 import lm
    none = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    assert lm.dispatch(torch.empty(0, 16, device="cuda"), none).shape == (0, 16)
    assert lm.combine(torch.empty(5, 16, device="cuda"), none).shape == (0, 16)
    lost = torch.full((4, 3), -1, dtype=torch.int32, device="cuda")
    assert (lm.combine(torch.empty(0, 16, device="cuda"), lost) == 0).all()
    dy, dw = lm.combine_grad(torch.ones(4, 16, device="cuda"), torch.empty(0, 16, device="cuda"), lost, torch.ones(4, 3, device="cuda"))
    assert dy.shape == (0, 16) and (dw == 0).all()


def test_refusals(cuda):
    from bafe_b200 import lm
    x, place, w = torch.randn(4, 16, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.ones(4, 2, device="cuda")
    y = torch.randn(8, 16, device="cuda")
    for call in (lambda: lm.dispatch(x, place.long()), lambda: lm.dispatch(x, place[:3]), lambda: lm.dispatch(x, place[0]),
                 lambda: lm.dispatch(x, place, out=torch.empty(8, 15, device="cuda")),
                 lambda: lm.dispatch(x, place, out=x), lambda: lm.dispatch(x, place, scale_out=w[0]),
                 lambda: lm.dispatch(x, place, scale=w[:, 0].half()),
                 lambda: lm.dispatch(x, place[:1].expand(4, 2)),
                 lambda: lm.combine(y, place, w.half()), lambda: lm.combine(y, place, w[:, :1]),
                 lambda: lm.combine(y, place, out=y[:4]), lambda: lm.combine(y, place, out=torch.empty(4, 16, device="cuda").half()),
                 lambda: lm.combine_grad(x, y, place, None), lambda: lm.combine_grad(x[:, :15], y, place, w),
                 lambda: lm.combine_grad(x.half(), y, place, w), lambda: lm.combine_grad(x, y, place, w, out=x),
                 lambda: lm.combine_grad(x, y, place, w, weight_out=w), lambda: lm.combine(y.requires_grad_(), place),
                 lambda: lm.dispatch(x.cpu(), place)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        lm.combine(y.detach().double(), place)
