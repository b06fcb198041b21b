"""The routing and loss operators together with the ones they stand beside, as a
model uses them: a block of routed experts with an output loss, forward and
all gradients (norm, router, dispatch, grouped product, combine, norm, loss),
eager and as one captured graph, against the same in 64 bits; and the same
calls on two streams at once, on padded rows, and beside torch's autograd.

Tolerances.  2-norms: a rounding to bf16 is below 2^-9 of a vector's 2-norm
(half a step at most, evenly spread), a later product carries an earlier
relative error through; the square root of the number of rounded stages times
2^-9 bounds the expected error and twice as much is allowed.  The choice of
experts is compared bit for bit where its logits are given in 32 bits; in the
chain both sides use the experts that the router chose.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -9


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, seed, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def rel(got, want):
    return float((got.double() - want).norm() / want.norm())


class Block:
    """h = x; n = norm(h); route; y = experts(n); h2 = h + combine; loss(norm(h2) W)."""

    def __init__(self, rows, width, experts, k, vocab, seed=0, padded=0):
        self.k, self.rows = k, rows
        self.x = randn((rows, width), seed + 1)
        self.g1, self.g2 = (1 + 0.1 * randn((width,), seed + 2)).bfloat16(), (1 + 0.1 * randn((width,), seed + 3)).bfloat16()
        self.router = randn((width, experts), seed + 4, width ** -0.5, torch.float32)
        self.w = randn((experts, width, width), seed + 5, width ** -0.5)
        self.out = randn((vocab, width), seed + 6, 2.0 * width ** -0.5)
        self.target = torch.randint(0, vocab, (rows,), generator=gen(seed + 7), device="cuda")
        self.bias = 0.05 * randn((experts,), seed + 8, 1.0, torch.float32)
        self.pad = torch.zeros(rows, dtype=torch.bool, device="cuda")
        if padded:
            self.pad[-padded:] = True
            self.target[self.pad] = -100

    def forward(self, lm, stream=None):
        n, h = lm.rms_norm(self.x, self.g1, self.x, stream=stream)
        logits = (n.float() @ self.router).masked_fill(self.pad[:, None], -math.inf)
        r = lm.route(logits, self.k, score="sigmoid", bias=self.bias, groups=2, keep_groups=1, scale=2.0, stream=stream)
        xs = lm.dispatch(n, r.place, stream=stream)
        ys = lm.grouped_matmul(xs, self.w, r.offsets, stream=stream)
        c = lm.combine(ys, r.place, r.weights, stream=stream)
        n2, h2 = lm.rms_norm(c, self.g2, h, stream=stream)
        loss, lse = lm.linear_cross_entropy(n2, self.out, self.target, stream=stream)
        return n, h, logits, r, xs, ys, c, n2, h2, loss, lse

    def backward(self, lm, kept, dloss, stream=None):
        n, h, logits, r, xs, ys, c, n2, h2, loss, lse = kept
        dn2, dout = lm.linear_cross_entropy_grad(dloss, n2, self.out, self.target, lse, stream=stream)
        dh2, dg2 = lm.rms_norm_grad(dn2, h2, self.g2, stream=stream)
        dys, dweights = lm.combine_grad(dh2, ys, r.place, r.weights, stream=stream)
        dxs = lm.grouped_matmul_grad_input(dys, self.w, r.offsets, stream=stream)
        dw = lm.grouped_matmul_grad_weight(dys, xs, r.offsets, stream=stream)
        dn = lm.combine(dxs, r.place, stream=stream)
        dlogits = lm.route_grad(dweights, logits, r.experts, score="sigmoid", scale=2.0, stream=stream)
        dn = dn + (dlogits @ self.router.t()).to(dn.dtype)
        dx, dg1 = lm.rms_norm_grad(dn, h, self.g1, dh2, stream=stream)
        return dout, dg2, dw, dlogits, dx, dg1

    def step(self, lm, dloss, stream=None):
        kept = self.forward(lm, stream)
        return (kept[9], kept[8], kept[3].experts) + self.backward(lm, kept, dloss, stream)


def reference(b, experts, dloss):
    """64 bits, torch's differentiation, with the given choice."""
    x = b.x.double().requires_grad_()
    g1, g2, w, out, router = (t.double().requires_grad_() for t in (b.g1, b.g2, b.w, b.out, b.router))
    h = x + b.x.double()                                 # the gradient of x alone, as of a residual
    n = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * g1
    logits = n @ router
    logits.retain_grad()
    some = experts >= 0
    at = experts.long().clamp_min(0)
    s = torch.sigmoid(logits).gather(1, at) * some
    weights = 2.0 * s / s.sum(-1, keepdim=True).clamp_min(1e-300)
    c = torch.zeros_like(h)
    for e in range(w.shape[0]):
        y = n @ w[e].t()
        c = c + y * (weights * (at == e) * some).sum(-1, keepdim=True)
    h2 = h + c
    n2 = h2 / torch.sqrt(h2.square().mean(-1, keepdim=True) + 1e-6) * g2
    z = n2 @ out.t()
    counts = b.target != -100
    loss = (torch.logsumexp(z, -1) - z.gather(1, b.target.clamp_min(0)[:, None])[:, 0]) * counts
    (loss * dloss.double()).sum().backward()
    return loss.detach(), h2.detach(), out.grad, g2.grad, w.grad, logits.grad, x.grad, g1.grad


@pytest.mark.parametrize("padded", [0, 37])
def test_training_step(cuda, padded):
    import bafe_b200
    from bafe_b200 import lm
    b = Block(300, 256, 12, 3, 1003, padded=padded)
    dloss = torch.full((1,), 1.0 / 300, device="cuda").expand(300)
    eager = b.step(lm, dloss)
    bafe_b200.synchronize()
    want = reference(b, eager[2], dloss)
    if padded:
        assert (eager[2][b.pad] == -1).all() and (eager[2][~b.pad] >= 0).all()
        assert (eager[0][b.pad] == 0).all()
    # rounded stages before each: h, n, xs-products (ys), c, h2, n2 ... and back
    limits = dict(loss=None, h2=4, dout=7, dg2=8, dw=10, dlogits=10, dx=12, dg1=12)
    for name, got, ref in zip(limits, (eager[0], eager[1]) + eager[3:], want):
        if name == "loss":
            assert float((got.double() - ref).abs().max()) < 0.1     # logits of size 2 sqrt(width) n w off by 6 roundings
            continue
        assert torch.isfinite(got).all(), name
        assert rel(got, ref) < 2 * HALF * limits[name] ** 0.5, (name, rel(got, ref))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = b.step(lm, dloss)
    for _ in range(2):
        graph.replay()
    bafe_b200.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(captured, eager))
    # the same graph on other rows, targets and routes; every second target is ignored
    b.x.copy_(randn((300, 256), 77))
    b.target[::2] = -100
    graph.replay()
    again = b.step(lm, dloss)
    bafe_b200.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(captured, again))
    assert (captured[0][::2] == 0).all()


def test_steps_on_two_streams_at_once(cuda):
    from bafe_b200 import lm
    blocks = [Block(257, 128, 8, 2, 515, seed=100 * i) for i in range(2)]
    dloss = torch.rand(257, generator=gen(5), device="cuda")
    want = [b.step(lm, dloss) for b in blocks]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        got = []
        for b, s in zip(blocks, streams):
            with torch.cuda.stream(s):                   # torch's own products between the calls run there too
                got.append(b.step(lm, dloss, s))
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(p, q))


def test_calls_on_another_stream_than_the_current_one(cuda):
    from bafe_b200 import lm
    side = torch.cuda.Stream()
    z, bias = randn((500, 64), 1, 1.0, torch.float32), randn((64,), 2, 0.1, torch.float32)
    x, w, t = randn((500, 96), 3), randn((700, 96), 4, 0.2), torch.randint(0, 700, (500,), generator=gen(5), device="cuda")
    want_r = lm.route(z, 4, score="sigmoid", bias=bias)
    want_l = lm.linear_cross_entropy(x, w, t)
    want_g = lm.linear_cross_entropy_grad(want_l[0], x, w, t, want_l[1])
    want_y = lm.dispatch(x, want_r.place)
    torch.cuda.synchronize()
    for _ in range(3):
        r = lm.route(z, 4, score="sigmoid", bias=bias, stream=side)
        y = lm.dispatch(x, r.place, stream=side)
        c = lm.combine(y, r.place, r.weights, stream=side)
        l = lm.linear_cross_entropy(x, w, t, stream=side)
        g = lm.linear_cross_entropy_grad(l[0], x, w, t, l[1], stream=side)
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(r, want_r)) and torch.equal(y, want_y)
        assert all(torch.equal(p, q) for p, q in zip(l + g, want_l + want_g))
        assert torch.equal(c, lm.combine(want_y, want_r.place, want_r.weights))
    with pytest.raises(TypeError):
        lm.route(z, 4, stream=side.cuda_stream)


def test_two_graphs_of_the_same_calls(cuda):
    """Scratch is each graph's own: replayed at once on two streams they give each its own results."""
    from bafe_b200 import lm
    sets = [(randn((5000, 200), 10 + i, 1.0, torch.float32), randn((300, 520), 20 + i), randn((3000, 520), 30 + i, 0.1),
             torch.randint(0, 3000, (300,), generator=gen(40 + i), device="cuda")) for i in range(2)]
    dloss = torch.rand(300, generator=gen(50), device="cuda")

    def calls(z, x, w, t):
        r = lm.route(z, 5, score="sigmoid", groups=4, keep_groups=2)
        l, lse = lm.linear_cross_entropy(x, w, t)
        return tuple(r) + (l,) + lm.linear_cross_entropy_grad(dloss, x, w, t, lse)

    want = [calls(*s) for s in sets]
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(calls(*s))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(got, ref))


def test_beside_autograd(cuda):
    """From a torch.autograd.Function, whose gradients reach the calls as autograd makes them (expanded, of the mean)."""
    from bafe_b200 import lm

    class Loss(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, t):
            loss, lse = lm.linear_cross_entropy(x, w, t)
            ctx.save_for_backward(x, w, t, lse)
            return loss

        @staticmethod
        def backward(ctx, dloss):
            x, w, t, lse = ctx.saved_tensors
            return lm.linear_cross_entropy_grad(dloss, x, w, t, lse) + (None,)

    x, w = randn((100, 64), 1).requires_grad_(), randn((333, 64), 2, 0.2).requires_grad_()
    t = torch.randint(0, 333, (100,), generator=gen(3), device="cuda")
    loss = Loss.apply(x, w, t).mean()
    loss.backward()
    x64, w64 = (v.detach().double().requires_grad_() for v in (x, w))
    ref = torch.nn.functional.cross_entropy(x64 @ w64.t(), t)
    ref.backward()
    assert abs(float(loss.detach()) - float(ref.detach())) < 1e-4
    assert rel(x.grad, x64.grad) < 2 * 2 ** 0.5 * HALF and rel(w.grad, w64.grad) < 2 * 2 ** 0.5 * HALF
    # out arguments tell autograd's graph that they were written
    out = torch.empty(100, 64, device="cuda").bfloat16()
    before = out._version
    with torch.no_grad():
        y = lm.linear_cross_entropy(x, w, t)
        lm.linear_cross_entropy_grad(y[0], x, w, t, y[1], out=out)
    assert out._version > before


def test_many_host_threads(cuda):
    """Several host threads on streams of their own, calls of different sizes: each gets its own results."""
    import threading
    from bafe_b200 import lm
    jobs = []
    for i, (rows, n) in enumerate(((3, 256), (700, 60), (2000, 300), (64, 8))):
        z = randn((rows, n), i, 1.0, torch.float32)
        x, w = randn((rows, 72), 10 + i), randn((n * 3, 72), 20 + i, 0.2)
        t = torch.randint(0, n * 3, (rows,), generator=gen(i), device="cuda")
        jobs.append((z, x, w, t))

    def run(j, stream):
        z, x, w, t = j
        r = lm.route(z, 3, stream=stream)
        y = lm.dispatch(x, r.place, stream=stream)
        l, lse = lm.linear_cross_entropy(x, w, t, stream=stream)
        return tuple(r) + (lm.combine(y, r.place, r.weights, stream=stream), l, lse) + \
            lm.linear_cross_entropy_grad(l, x, w, t, lse, stream=stream)

    want = [run(j, None) for j in jobs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        for _ in range(15):
            got = run(jobs[i], s)
            s.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad
