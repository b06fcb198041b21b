"""The operators together, as a model uses them: an expert feed-forward block
in training (norm, grouped product, and all gradients, chained) and a decode
step (norm to 8 bits, grouped 8-bit product, norm, 4-bit projection), eager
and as one captured graph, against the same chain in 64 bits.

Tolerances.  The chains are compared in the 2-norm.  A rounding is off by at
most half a step (2^-8 for bf16, 2^-4 for e4m3), evenly spread, so its
2-norm is below 2^-8 / sqrt(3) < 2^-9 and 2^-4 / sqrt(3); the 32-bit errors
are far below.  A later product carries an earlier stage's relative error
through as it is, for errors of independent signs: the square root of the
number of rounded stages times that bounds the expected error, and twice as
much is allowed.
"""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, seed, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def rel(got, want):
    return float((got.double() - want).norm() / want.norm())


def norm64(x, w, res):
    h = x.double() + res.double()
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w.double(), h


def test_expert_block_training_step(cuda):
    """y = experts(norm(x + res)); loss = sum(y * c) + sum(h * d): every gradient, in one run of calls."""
    import bafe_b200
    from bafe_b200 import lm
    sizes, width, inner = [100, 0, 37, 250, 1], 384, 520
    rows = sum(sizes)
    off = torch.tensor(list(itertools.accumulate([0] + sizes)), dtype=torch.int32, device="cuda")
    x, res, g = randn((rows, width), 1), randn((rows, width), 2, 2.0), (1 + 0.1 * randn((width,), 3)).to(torch.bfloat16)
    w = randn((5, inner, width), 4, width ** -0.5)
    c, d = randn((rows, inner), 5, 0.1), randn((rows, width), 6, 0.1)

    def step():
        n, h = lm.rms_norm(x, g, res)
        y = lm.grouped_matmul(n, w, off)
        dn = lm.grouped_matmul_grad_input(c, w, off)
        dw = lm.grouped_matmul_grad_weight(c, n, off)
        dx, dg = lm.rms_norm_grad(dn, h, g, d)
        return n, h, y, dn, dw, dx, dg

    eager = step()
    bafe_b200.synchronize()
    # 64 bits, through torch's own differentiation
    x64, w64, g64 = (t.double().requires_grad_() for t in (x, w, g))
    h64 = x64 + res.double()
    n64 = h64 / torch.sqrt(h64.square().mean(-1, keepdim=True) + 1e-6) * g64
    parts, at = [], 0
    for e, z in enumerate(sizes):
        parts.append(n64[at:at + z] @ w64[e].t())
        at += z
    y64 = torch.cat(parts)
    ((y64 * c.double()).sum() + (h64 * d.double()).sum()).backward()
    half = 2.0 ** -9
    assert rel(eager[2], y64.detach()) < 2 * half * 3 ** 0.5          # h, n, y
    assert rel(eager[4], w64.grad) < 2 * half * 3 ** 0.5              # h, n, dw
    assert rel(eager[5], x64.grad) < 2 * half * 3 ** 0.5              # h, dn, dx
    assert rel(eager[6], g64.grad) < 2 * half * 3 ** 0.5              # h, dn, dg
    assert (eager[4][1] == 0).all()

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(2):
        graph.replay()
    bafe_b200.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, eager))
    # the same graph on other rows and other group sizes
    x.copy_(randn((rows, width), 7))
    off.copy_(torch.tensor([0, 0, 200, 200, 388, 388], dtype=torch.int32))
    graph.replay()
    again = step()
    bafe_b200.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, again))


def test_decode_step(cuda):
    """Norm to 8 bits -> 8-bit experts -> norm to 8 bits -> 4-bit projection of 8-bit rows, and of 16-bit ones."""
    import bafe_b200
    from bafe_b200 import lm
    rows, width, vocab, group = 6, 512, 1000, 128
    off = torch.tensor([0, 2, 2, 5, 6], dtype=torch.int32, device="cuda")
    owner = [0, 0, 2, 2, 2, 3]
    x, res = randn((rows, width), 11), randn((rows, width), 12, 2.0)
    g1, g2 = (1 + 0.1 * randn((width,), 13)).to(torch.bfloat16), (1 + 0.1 * randn((width,), 14)).to(torch.bfloat16)
    w = randn((4, width, width), 15, 1.0, torch.float32)
    ws = w.abs().amax(-1) / 448.0
    w8 = (w / ws[..., None]).to(torch.float8_e4m3fn)
    q = torch.randint(0, 256, (vocab, width // 2), generator=gen(16), device="cuda", dtype=torch.uint8)
    s = (0.01 + 0.01 * torch.rand(vocab, width // group, generator=gen(17), device="cuda")).to(torch.bfloat16)
    z = torch.randint(0, 16, (vocab, width // group), generator=gen(18), device="cuda", dtype=torch.uint8)

    def step():
        a, a_scale, h = lm.rms_norm_e4m3(x, g1, res)
        y = lm.grouped_matmul(a, w8, off, x_scale=a_scale, w_scale=ws)
        b, b_scale, h2 = lm.rms_norm_e4m3(y, g2, h)
        n, _ = lm.rms_norm(y, g2, h)
        return (lm.matvec_w4(b, q, s, z, group=group, x_scale=b_scale), lm.matvec_w4(n, q, s, z, group=group), h2)

    eager = step()
    bafe_b200.synchronize()
    n1, h = norm64(x, g1, res)
    y = torch.stack([n1[i] @ (w8[e].double() * ws[e].double()[:, None]).t() for i, e in enumerate(owner)])
    n2, h2 = norm64(y, g2, h)
    at = torch.arange(width, device="cuda")
    v = ((q[:, at // 2].int() >> (4 * (at % 2)).int()) & 15).double()
    w4 = (v - z[:, at // group].double()) * s[:, at // group].double()
    want = n2 @ w4.t()
    assert rel(eager[0], want) < 2 * 2.0 ** -4 * 2 ** 0.5       # two roundings to 8 bits lead
    assert rel(eager[1], want) < 2 * 2.0 ** -4                  # one
    assert rel(eager[2], h2) < 2 * 2.0 ** -4

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    bafe_b200.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, eager))


def test_calls_on_two_streams_at_once(cuda):
    """The same calls on two streams, with scratch of their own, give the bits of one after the other."""
    from bafe_b200 import lm
    off = torch.tensor([0, 70, 201], dtype=torch.int32, device="cuda")
    sets = [(randn((201, 333), 21 + i), randn((333,), 31 + i), randn((2, 222, 333), 41 + i, 0.1)) for i in range(2)]
    q = torch.randint(0, 256, (64, 4096), generator=gen(5), device="cuda", dtype=torch.uint8)
    s = randn((64, 64), 6)
    xs = [randn((5, 8192), 51 + i) for i in range(2)]

    def run(i, stream=None):
        x, g, w = sets[i]
        n = lm.rms_norm(x, g, stream=stream)
        y = lm.grouped_matmul(n, w, off, stream=stream)
        dw = lm.grouped_matmul_grad_weight(y, n, off, stream=stream)
        dx, dg = lm.rms_norm_grad(n, x, g, stream=stream)
        return y, dw, dx, dg, lm.matvec_w4(xs[i], q, s, stream=stream)

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = [run(i, streams[i]) for i in range(2)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
