"""The language-model operators beside torch's autograd: a gradient that a
call would drop is refused, an output written in place is seen by the graph
that saved it, and a torch.autograd.Function around them differentiates."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def randn(*shape, seed=1, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def calls():
    """Each entry point with its floating-point operands, as (call, operands)."""
    from bafe_b200 import lm
    x, g, w = randn(12, 64), randn(64, seed=2), randn(2, 32, 64, seed=3)
    dy, off = randn(12, 32, seed=4), torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda")
    q = torch.randint(0, 256, (32, 32), device="cuda", dtype=torch.uint8)
    s, xs = randn(32, 2, seed=5), torch.ones(12, device="cuda")
    return [(lm.rms_norm, [x, g, x.clone()]), (lm.rms_norm_e4m3, [x, g, x.clone()]),
            (lm.rms_norm_grad, [randn(12, 64, seed=6), x, g, randn(12, 64, seed=7)]),
            (lambda a, b: lm.grouped_matmul(a, b, off), [x, w]),
            (lambda a, b, c, d: lm.grouped_matmul(a.detach().to(torch.float8_e4m3fn), b.detach().to(torch.float8_e4m3fn),
                                                  off, x_scale=c, w_scale=d), [x, w, xs, torch.ones(2, 32, device="cuda")]),
            (lambda a, b: lm.grouped_matmul_grad_input(a, b, off), [dy, w]),
            (lambda a, b: lm.grouped_matmul_grad_weight(a, b, off), [dy, x]),
            (lambda a, b: lm.matvec_w4(a, q, b, group=32), [x, s]),
            (lambda a, b, c: lm.matvec_w4(a.detach().to(torch.float8_e4m3fn), q, b, group=32, x_scale=c), [x, s, xs])]


def test_a_gradient_that_would_be_lost_is_refused(cuda):
    for n, (call, operands) in enumerate(calls()):
        want = call(*operands)
        for i in range(len(operands)):
            if n in (4, 8) and i < (2 if n == 4 else 1):
                continue                                 # detached on the way to 8 bits
            some = [t.clone().requires_grad_(j == i) for j, t in enumerate(operands)]
            with pytest.raises(ValueError, match="gradient"):
                call(*some)
            with torch.no_grad():
                got = call(*some)
            for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                assert not a.requires_grad and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_outputs_of_a_leaf_are_refused(cuda):
    from bafe_b200 import lm
    x, g = randn(12, 64), randn(64, seed=2)
    leaf = torch.empty(12, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        lm.rms_norm(x, g, out=leaf)
    with pytest.raises(ValueError, match="gradient"):
        lm.rms_norm(x, g, x, residual_out=leaf)
    with torch.no_grad():
        assert lm.rms_norm(x, g, out=leaf) is leaf


def test_a_graph_sees_what_was_overwritten(cuda):
    from bafe_b200 import lm
    g, off = randn(64, seed=2), torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda")
    w = randn(2, 64, 64, seed=3)
    q, s = torch.randint(0, 256, (64, 32), device="cuda", dtype=torch.uint8), randn(64, 2, seed=5)
    x, h = randn(12, 64), randn(12, 64, seed=8)
    f32 = torch.ones(12, device="cuda")
    writes = [(randn(12, 64), lambda t: lm.rms_norm(t, g, out=t)),
              (randn(12, 64), lambda t: lm.rms_norm(x, g, t, residual_out=t)),
              (f32, lambda t: lm.rms_norm_e4m3(x, g, scale_out=t)),
              (randn(12, 64), lambda t: lm.rms_norm_grad(t, h, g, out=t)),
              (randn(64), lambda t: lm.rms_norm_grad(x, h, g, weight_out=t)),
              (randn(12, 64), lambda t: lm.grouped_matmul(x, w, off, out=t)),
              (randn(12, 64), lambda t: lm.grouped_matmul_grad_input(x, w, off, out=t)),
              (randn(2, 64, 64), lambda t: lm.grouped_matmul_grad_weight(x, h, off, out=t)),
              (randn(12, 64), lambda t: lm.matvec_w4(x, q, s, group=32, out=t))]
    for t, write in writes:
        scale = torch.ones((), device="cuda", requires_grad=True)
        kept = t * scale.to(t.dtype)                     # saves t
        version = t._version
        write(t)
        assert t._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.sum().backward()


def test_function_of_the_callers(cuda):
    """Forward and backward as explicit calls inside a torch.autograd.Function, against torch's own differentiation in 64 bits."""
    from bafe_b200 import lm

    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            ctx.save_for_backward(x, w)
            return lm.rms_norm(x, w)

        @staticmethod
        def backward(ctx, dy):
            x, w = ctx.saved_tensors
            return lm.rms_norm_grad(dy.contiguous(), x, w)

    x, w, c = randn(20, 96, dtype=torch.float32), randn(96, seed=2, dtype=torch.float32), randn(20, 96, seed=3, dtype=torch.float32)
    x.requires_grad_()
    w.requires_grad_()
    (Norm.apply(x, w) * c).sum().backward()
    x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    (x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + 1e-6) * w64 * c.double()).sum().backward()
    # 2^-17 relative to the terms that cancel, as in test_gpu_lm_norm.py
    assert float((x.grad.double() - x64.grad).abs().max()) <= 2.0 ** -17 * 4 * float(x64.grad.abs().max() + 1)
    assert float((w.grad.double() - w64.grad).abs().max()) <= 2.0 ** -17 * 20 * float(w64.grad.abs().max() + 1)
