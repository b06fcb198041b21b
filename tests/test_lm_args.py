"""The language-model operators' refusals that need no GPU: arguments are
checked before a device is asked for, in the C entries and in Python."""
import ctypes

import pytest
import torch

from bafe_b200 import _binding, lm
from bafe_b200._binding import DTYPE_BF16, DTYPE_E4M3, DTYPE_F32, lib

P = ctypes.c_void_p(256)        # never dereferenced: every call below is refused


def message():
    code, msg = _binding.last_error()
    return code, msg


def norm(x=P, x_ld=64, res=None, res_ld=0, w=P, y=P, y_ld=64, scale=None, h=None, h_ld=0, rows=4, width=64,
         dtype=DTYPE_BF16, wdtype=DTYPE_BF16, ydtype=DTYPE_BF16, eps=1e-6):
    return lib.bafe_cuda_rms_norm(x, x_ld, res, res_ld, w, y, y_ld, scale, h, h_ld, rows, width, dtype, wdtype, ydtype,
                                  eps, None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(w=None), dict(y=None), dict(x_ld=63), dict(y_ld=1), dict(rows=-1), dict(width=0),
    dict(width=1 << 31), dict(dtype=1), dict(dtype=DTYPE_E4M3), dict(wdtype=4), dict(ydtype=DTYPE_F32),
    dict(ydtype=DTYPE_E4M3), dict(res=P, res_ld=64), dict(h=P, h_ld=64), dict(res=P, res_ld=3, h=P, h_ld=64),
    dict(eps=-1.0), dict(eps=float("nan")),
])
def test_norm_entry_refuses(bad):
    assert norm(**bad) == 8
    code, msg = message()
    assert code == 8 and "rms_norm" in msg


def test_norm_entry_without_rows():
    assert norm(rows=0, x=None, y=None) == 0


def test_norm_grad_entry_refuses():
    def call(dy=P, h=P, w=P, dx=P, dw=P, rows=4, width=64, dy_ld=64, dtype=DTYPE_BF16, dh=None, dh_ld=0):
        return lib.bafe_cuda_rms_norm_grad(dy, dy_ld, h, 64, w, dh, dh_ld, dx, 64, dw, rows, width, dtype, dtype, 1e-6,
                                           None, 0, None)
    for bad in (dict(dy=None), dict(h=None), dict(w=None), dict(dx=None), dict(dw=None), dict(rows=-2), dict(width=0),
                dict(dy_ld=10), dict(dtype=2), dict(dh=P, dh_ld=5)):
        assert call(**bad) == 8, bad
    assert lib.bafe_cuda_rms_norm_grad_workspace(-1, 64, DTYPE_BF16) == -1
    assert lib.bafe_cuda_rms_norm_grad_workspace(4, 64, DTYPE_E4M3) == -1


def test_python_refuses_cpu_tensors():
    x, w = torch.zeros(4, 64), torch.ones(64)
    for call in (lambda: lm.rms_norm(x, w), lambda: lm.rms_norm_e4m3(x, w), lambda: lm.rms_norm_grad(x, x, w)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        lm.rms_norm([1.0], w)


def test_w4_entry_refuses():
    def call(x=P, x_ld=256, q=P, q_ld=128, s=P, s_ld=2, z=None, z_ld=0, y=P, y_ld=32, tokens=2, n=32, k=256, group=128,
             xt=DTYPE_BF16, st=DTYPE_BF16, yt=DTYPE_BF16):
        return lib.bafe_cuda_matvec_w4(x, x_ld, None, q, q_ld, s, s_ld, z, z_ld, y, y_ld, tokens, n, k, group, xt, st, yt,
                                       None, 0, None)
    for bad in (dict(x=None), dict(q=None), dict(s=None), dict(y=None), dict(x_ld=255), dict(q_ld=127), dict(s_ld=1),
                dict(z=P, z_ld=1), dict(y_ld=31), dict(tokens=-1), dict(n=-1), dict(k=0), dict(k=1 << 23),
                dict(group=0), dict(group=48), dict(group=-32), dict(xt=DTYPE_F32), dict(st=2), dict(yt=DTYPE_F32),
                dict(yt=DTYPE_E4M3)):
        assert call(**bad) == 8, bad
        assert "matvec_w4" in message()[1]
    assert call(tokens=0, x=None, y=None) == 0
    assert lib.bafe_cuda_matvec_w4_workspace(1, 32, 256, 33) == -1
    with pytest.raises(ValueError, match="CUDA"):
        lm.matvec_w4(torch.zeros(1, 64, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1))


def test_grouped_entries_refuse():
    def call(x=P, x_ld=64, w=P, w_ld=64, w_stride=64 * 32, kmajor=1, off=P, xs=None, ws=None, ws_ld=0, y=P, y_ld=32,
             rows=8, experts=4, n=32, k=64, dt=DTYPE_BF16, yt=DTYPE_BF16):
        return lib.bafe_cuda_grouped_matmul(x, x_ld, w, w_ld, w_stride, kmajor, off, xs, ws, ws_ld, y, y_ld, rows, experts,
                                            n, k, dt, yt, None, 0, None)
    for bad in (dict(x=None), dict(w=None), dict(off=None), dict(y=None), dict(x_ld=63), dict(w_ld=63), dict(w_stride=9),
                dict(y_ld=31), dict(rows=-1), dict(experts=0), dict(experts=1025), dict(n=0), dict(k=0),
                dict(dt=DTYPE_F32), dict(yt=DTYPE_F32), dict(yt=4), dict(xs=P), dict(ws=P),
                dict(dt=DTYPE_E4M3), dict(dt=DTYPE_E4M3, xs=P, ws=P, ws_ld=31),
                dict(dt=DTYPE_E4M3, xs=P, ws=P, ws_ld=32, kmajor=0),
                dict(k=63, x_ld=63, w_ld=63)):          # unaligned rows without a workspace
        assert call(**bad) == 8, bad
        assert "grouped_matmul" in message()[1]
    assert call(rows=0, x=None, y=None) == 0
    assert lib.bafe_cuda_grouped_matmul_workspace(P, 64, P, 64, 2048, 1, 8, 4, 32, 64, DTYPE_BF16) == 0
    assert lib.bafe_cuda_grouped_matmul_workspace(P, 63, P, 64, 2048, 1, 8, 4, 32, 63, DTYPE_BF16) == 8 * 64 * 2
    assert lib.bafe_cuda_grouped_matmul_workspace(P, 64, P, 64, 2048, 1, 8, 0, 32, 64, DTYPE_BF16) == -1

    def grad(dy=P, dy_ld=32, x=P, x_ld=64, off=P, dw=P, dw_ld=64, dw_stride=2048, rows=8, experts=4, n=32, k=64,
             dt=DTYPE_BF16):
        return lib.bafe_cuda_grouped_matmul_grad_weight(dy, dy_ld, x, x_ld, off, dw, dw_ld, dw_stride, rows, experts, n, k,
                                                        dt, None, 0, None)
    for bad in (dict(dy=None), dict(x=None), dict(off=None), dict(dw=None), dict(dy_ld=1), dict(x_ld=1), dict(dw_ld=1),
                dict(dw_stride=1), dict(rows=-1), dict(experts=0), dict(n=0), dict(k=0), dict(dt=DTYPE_F32),
                dict(dt=DTYPE_E4M3)):
        assert grad(**bad) == 8, bad
    h = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: lm.grouped_matmul(h, torch.zeros(2, 8, 64), torch.zeros(3, dtype=torch.int32)),
                 lambda: lm.grouped_matmul_grad_input(h, torch.zeros(2, 64, 8), torch.zeros(3, dtype=torch.int32)),
                 lambda: lm.grouped_matmul_grad_weight(h, h, torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_operands_side_by_side_do_not_overlap():
    """Columns of one buffer are apart; shifted rows, and columns that meet, are not."""
    buf = torch.zeros(8, 100)
    a, b, c = buf[:, :40], buf[:, 40:80], buf[:, 30:70]
    assert not lm._overlap(a, b) and not lm._overlap(b, a)
    assert lm._overlap(a, c) and lm._overlap(c, a) and lm._overlap(b, c)
    assert lm._overlap(buf[:4], buf[3:]) and not lm._overlap(buf[:4], buf[4:])
    assert lm._overlap(buf[:-1], buf[1:])
    assert lm._overlap(buf[:, 60:], buf[1:, :1].expand(7, 1)[:, :1]) is False
    assert lm._overlap(a, buf.view(-1)[10:300])
    assert not lm._overlap(buf[:0], buf)


def test_entries_refuse_pointers_inside_an_element():
    odd, half = ctypes.c_void_p(257), ctypes.c_void_p(258)
    for bad in (dict(x=odd), dict(w=odd), dict(y=odd), dict(res=odd, res_ld=64, h=P, h_ld=64),
                dict(res=P, res_ld=64, h=odd, h_ld=64), dict(w=half, wdtype=DTYPE_F32),
                dict(x=half, dtype=DTYPE_F32, wdtype=DTYPE_F32, ydtype=DTYPE_F32)):
        assert norm(**bad) == 8, bad
        assert "element's size" in message()[1]
    for at in range(4):
        p = [P] * 4
        p[at] = odd
        assert lib.bafe_cuda_rms_norm_grad(p[0], 64, p[1], 64, p[2], None, 0, p[3], 64, P, 4, 64, DTYPE_BF16, DTYPE_BF16,
                                           1e-6, P, 1 << 30, None) == 8
        assert "element's size" in message()[1]
    for x, s, y, st in ((odd, P, P, DTYPE_BF16), (P, odd, P, DTYPE_BF16), (P, P, odd, DTYPE_BF16), (P, half, P, DTYPE_F32)):
        assert lib.bafe_cuda_matvec_w4(x, 256, None, P, 128, s, 2, None, 0, y, 32, 2, 32, 256, 128, DTYPE_BF16, st,
                                       DTYPE_BF16, None, 0, None) == 8
        assert "element's size" in message()[1]
    for x, w, off, y in ((odd, P, P, P), (P, odd, P, P), (P, P, half, P), (P, P, P, odd)):
        assert lib.bafe_cuda_grouped_matmul(x, 64, w, 64, 2048, 1, off, None, None, 0, y, 32, 8, 4, 32, 64, DTYPE_BF16,
                                            DTYPE_BF16, P, 1 << 30, None) == 8
        assert "element's size" in message()[1]
        assert lib.bafe_cuda_grouped_matmul_grad_weight(x, 32, w, 64, off, y, 64, 2048, 8, 4, 32, 64, DTYPE_BF16, P,
                                                        1 << 30, None) == 8
        assert "element's size" in message()[1]


def test_route_entries_refuse():
    def call(z=P, ld=64, bias=None, w=P, e=P, off=P, place=P, rows=80, n=64, k=4, groups=1, keep=1, top=2, score=0,
             scale=1.0, dt=DTYPE_F32, ws=P, need=1 << 30):
        return lib.bafe_cuda_route(z, ld, bias, w, e, off, place, rows, n, k, groups, keep, top, score, 1, scale, dt, ws,
                                   need, None)
    odd = ctypes.c_void_p(258)
    for bad in (dict(z=None), dict(w=None), dict(e=None), dict(off=None), dict(place=None), dict(ld=63), dict(rows=-1),
                dict(n=0), dict(n=1025), dict(k=0), dict(k=32), dict(n=3, k=4), dict(rows=1 << 29), dict(groups=0),
                dict(groups=3), dict(groups=64, keep=4), dict(groups=4, keep=5), dict(groups=4, keep=0),
                dict(groups=32, keep=1), dict(top=0), dict(top=3), dict(score=2), dict(score=-1),
                dict(scale=float("nan")), dict(scale=1e300), dict(dt=DTYPE_E4M3), dict(dt=2), dict(z=odd), dict(bias=odd),
                dict(off=odd)):
        assert call(**bad) == 8, bad
        assert "route" in message()[1]
    assert lib.bafe_cuda_route_workspace(-1, 64, 4) == -1
    assert lib.bafe_cuda_route_workspace(8, 64, 4) == 0

    def grad(dw=P, dw_ld=4, z=P, ld=64, e=P, e_ld=4, out=P, out_ld=64, rows=80, n=64, k=4, score=0, scale=1.0, dt=DTYPE_F32):
        return lib.bafe_cuda_route_grad(dw, dw_ld, z, ld, e, e_ld, out, out_ld, rows, n, k, score, 1, scale, dt, None)
    for bad in (dict(dw=None), dict(z=None), dict(e=None), dict(out=None), dict(dw_ld=-1), dict(ld=1), dict(e_ld=3),
                dict(out_ld=63), dict(k=65), dict(score=7), dict(dt=DTYPE_E4M3), dict(scale=float("inf")), dict(out=odd)):
        assert grad(**bad) == 8, bad
        assert "route_grad" in message()[1]
    assert grad(rows=0, dw=None) == 0
    z, e = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for f in (lambda: lm.route(z, 2), lambda: lm.route_grad(torch.zeros(4, 2), z, e)):
        with pytest.raises(ValueError, match="CUDA"):
            f()


def test_dispatch_entries_refuse():
    def move(x=P, x_ld=64, s=None, p=P, p_ld=4, y=P, y_ld=64, so=None, rows=8, k=4, n=32, width=64, es=2):
        return lib.bafe_cuda_dispatch(x, x_ld, s, p, p_ld, y, y_ld, so, rows, k, n, width, es, None)

    def total(y=P, y_ld=64, p=P, p_ld=4, w=P, w_ld=4, out=P, out_ld=64, rows=8, k=4, n=32, width=64, dt=DTYPE_BF16):
        return lib.bafe_cuda_combine(y, y_ld, p, p_ld, w, w_ld, out, out_ld, rows, k, n, width, dt, None)

    def grad(d=P, d_ld=64, y=P, y_ld=64, p=P, p_ld=4, w=P, w_ld=4, dy=P, dy_ld=64, dw=P, rows=8, k=4, n=32, width=64,
             dt=DTYPE_BF16):
        return lib.bafe_cuda_combine_grad(d, d_ld, y, y_ld, p, p_ld, w, w_ld, dy, dy_ld, dw, rows, k, n, width, dt, None)
    odd, half = ctypes.c_void_p(257), ctypes.c_void_p(258)
    sizes = (dict(rows=-1), dict(k=0), dict(k=32), dict(n=-1), dict(width=0), dict(width=1 << 31), dict(p_ld=3), dict(p=None),
             dict(p=half), dict(y=None), dict(y_ld=63), dict(y=odd))
    for bad in sizes + (dict(x=None), dict(x_ld=63), dict(s=P), dict(so=P), dict(es=3), dict(es=8), dict(x=odd),
                        dict(s=half, so=P)):
        assert move(**bad) == 8, bad
        assert "dispatch" in message()[1]
    for bad in sizes + (dict(out=None), dict(out_ld=63), dict(w_ld=-1), dict(w=half), dict(out=odd), dict(dt=DTYPE_E4M3)):
        assert total(**bad) == 8, bad
        assert "combine" in message()[1]
    for bad in sizes + (dict(d=None), dict(d_ld=-1), dict(w=None), dict(dw=None), dict(dy=None), dict(dy_ld=63), dict(w_ld=-1),
                        dict(dw=half), dict(dy=odd), dict(dt=DTYPE_E4M3)):
        assert grad(**bad) == 8, bad
        assert "combine_grad" in message()[1]
    assert move(rows=0, x=None) == 0 and total(rows=0, y=None) == 0 and grad(rows=0, y=None) == 0
    x, p = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for f in (lambda: lm.dispatch(x, p), lambda: lm.combine(x, p), lambda: lm.combine_grad(x, x, p, torch.zeros(4, 2))):
        with pytest.raises(ValueError, match="CUDA"):
            f()


def test_loss_entries_refuse():
    def call(x=P, x_ld=64, w=P, w_ld=64, t=P, tb=8, loss=P, lse=P, rows=8, vocab=100, width=64, dt=DTYPE_BF16):
        return lib.bafe_cuda_linear_cross_entropy(x, x_ld, w, w_ld, t, tb, loss, lse, rows, vocab, width, -100, dt, None, 0,
                                                  None)

    def grad(dl=P, dl_ld=1, x=P, x_ld=64, w=P, w_ld=64, t=P, tb=8, lse=P, dx=P, dx_ld=64, dw=P, dw_ld=64, rows=8, vocab=100,
             width=64, dt=DTYPE_BF16):
        return lib.bafe_cuda_linear_cross_entropy_grad(dl, dl_ld, x, x_ld, w, w_ld, t, tb, lse, dx, dx_ld, dw, dw_ld, rows,
                                                       vocab, width, -100, dt, None, 0, None)
    odd, half, four = ctypes.c_void_p(257), ctypes.c_void_p(258), ctypes.c_void_p(260)
    both = (dict(x=None), dict(w=None), dict(t=None), dict(x_ld=63), dict(w_ld=63), dict(tb=2), dict(rows=-1), dict(vocab=0),
            dict(width=0), dict(rows=1 << 25), dict(vocab=1 << 25), dict(width=1 << 21), dict(rows=1 << 24, vocab=1 << 24),
            dict(dt=DTYPE_F32), dict(dt=DTYPE_E4M3), dict(x=odd), dict(w=odd), dict(t=four), dict(lse=None), dict(lse=half))
    for bad in both + (dict(loss=None), dict(loss=half)):
        assert call(**bad) == 8, bad
        assert "linear_cross_entropy" in message()[1]
    for bad in both + (dict(dl=None), dict(dl_ld=-1), dict(dl=half), dict(dx=None), dict(dw=None), dict(dx_ld=63),
                       dict(dw_ld=63), dict(dx=odd), dict(dw=odd)):
        assert grad(**bad) == 8, bad
        assert "linear_cross_entropy_grad" in message()[1]
    assert call(rows=0, x=None) == 0
    assert lib.bafe_cuda_linear_cross_entropy_workspace(P, 64, P, 64, -1, 100, 64, 0) == -1
    assert lib.bafe_cuda_linear_cross_entropy_workspace(P, 64, P, 64, 0, 100, 64, 1) == 0
    x, t = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    for f in (lambda: lm.linear_cross_entropy(x, x, t), lambda: lm.linear_cross_entropy_grad(t, x, x, t, t)):
        with pytest.raises(ValueError, match="CUDA"):
            f()
