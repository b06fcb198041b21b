"""bafe_b200.lm -- operators of language models on device-resident tensors.

They stand beside the compiled graphs' matrix products, chains and
reductions and, like Kernel.run_torch, take torch CUDA tensors and only
enqueue on a CUDA stream:

    from bafe_b200 import lm

    y, h = lm.rms_norm(x, weight, residual)            # h = x + residual
    q, scale, h = lm.rms_norm_e4m3(x, weight, residual)
    dx, dweight = lm.rms_norm_grad(dy, h, weight, dh)
    y = lm.grouped_matmul(x, w, offsets)               # rows of x sorted by expert
    y = lm.grouped_matmul(q, w8, offsets, x_scale=scale, w_scale=w_scale)
    dx = lm.grouped_matmul_grad_input(dy, w, offsets)
    dw = lm.grouped_matmul_grad_weight(dy, x, offsets)
    y = lm.matvec_w4(x, qweight, scales, zeros, group=128)
    weights, experts, offsets, place = lm.route(logits, k)   # a router's choice, and the order by expert
    xs = lm.dispatch(x, place)                         # rows sorted by expert, for grouped_matmul
    out = lm.combine(ys, place, weights)               # and back
    dys, dweights = lm.combine_grad(dout, ys, place, weights)
    dx = lm.combine(dxs, place)                        # gradient of dispatch
    dlogits = lm.route_grad(dweights, logits, experts)
    loss, lse = lm.linear_cross_entropy(x, w, target)  # of the logits x @ w.T, which are not kept
    dx, dw = lm.linear_cross_entropy_grad(dloss, x, w, target, lse)

Common to all of them:
  * `stream` is a torch.cuda.Stream of the tensors' device (default: that
    device's current stream).  The call does not wait for other streams: the
    caller orders it after the work that fills its inputs.
  * Outputs and scratch are allocated on that stream (torch's allocator, so
    inside a graph capture they come from the graph's own pool); inputs that
    live on another stream are marked as used there.
  * `out` arguments are written in place and returned.
  * Unusable arguments raise ValueError or TypeError before anything is
    enqueued; a refused launch raises RuntimeError with the library's message.
  * No autograd: gradients are calls of their own, as every entry point of
    this package is explicit.  Where torch records gradients, tensors that
    require one are refused (their gradient would be lost); torch.no_grad()
    or a torch.autograd.Function of the caller's is the place for the call.
    Writing into `out` raises the tensor's version, so that a graph of
    torch's that saved it sees that it changed.
There is no CPU form: tensors elsewhere than on a CUDA device are refused.
"""
from __future__ import annotations

from operator import index
from typing import NamedTuple, Optional

import torch

from ._binding import DTYPE_BF16, DTYPE_E4M3, DTYPE_F16, DTYPE_F32, check, lib

_DTYPE = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16,
          torch.float8_e4m3fn: DTYPE_E4M3}
_ROW_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_HALF_TYPES = (torch.float16, torch.bfloat16)


class _Here:
    """The tensors' device and stream are the current ones: nothing to enter."""
    __slots__ = ()

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return None


class _There:
    """Makes the tensors' device and the call's stream current for its allocations."""
    __slots__ = ("_dev", "_stream")

    def __init__(self, index: int, stream):
        self._dev = torch.cuda.device(index)
        self._stream = None if stream is None else torch.cuda.stream(stream)

    def __enter__(self):
        self._dev.__enter__()
        if self._stream is not None:
            self._stream.__enter__()

    def __exit__(self, *exc):
        if self._stream is not None:
            self._stream.__exit__(*exc)
        self._dev.__exit__(*exc)


_HERE = _Here()
_current_device = torch._C._cuda_getDevice               # what torch.cuda.current_device reads
_current_raw_stream = torch._C._cuda_getCurrentRawStream


def _on(t: torch.Tensor, stream, tensors):
    """The call's cudaStream_t, and the context for its allocations and launch."""
    dev = t.get_device()
    if stream is None:
        return _current_raw_stream(dev), (_HERE if dev == _current_device() else _There(dev, None))
    if not isinstance(stream, torch.cuda.Stream):
        raise TypeError(f"stream must be a torch.cuda.Stream, got {type(stream).__name__}")
    if stream.device.index != dev:
        raise ValueError(f"stream of {stream.device} for tensors of {t.device}")
    raw = stream.cuda_stream
    if raw == _current_raw_stream(dev):
        return raw, (_HERE if dev == _current_device() else _There(dev, None))
    for x in tensors:
        if x is not None:
            x.record_stream(stream)
    return raw, _There(dev, stream)


def _explicit(*tensors) -> None:
    """Refuses tensors whose gradient this call would drop."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("a tensor requires a gradient, which these calls do not record: call the *_grad functions "
                                 "under torch.no_grad(), or from a torch.autograd.Function")


_written = torch._C._increment_version                   # of torch.autograd.graph.increment_version


def _cuda(name: str, t, like: Optional[torch.Tensor] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")


def _dense_last(name: str, t: torch.Tensor) -> None:
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")


def _ld(name: str, t: torch.Tensor) -> int:
    """Row stride of a 2-D tensor, in elements."""
    rows, width = t.shape
    ld, inner = t.stride()
    if inner != 1 and width > 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    if rows <= 1:
        return width
    if ld < width:
        raise ValueError(f"{name}'s rows overlap")
    return ld


def _rows(name: str, t: torch.Tensor, like: Optional[torch.Tensor] = None, types=None) -> int:
    """Checks a [rows, width] operand (of the same shape and type as `like`); its row stride."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _cuda(name, t)
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, got {tuple(t.shape)}")
    if like is None:
        if t.dtype not in types:
            raise TypeError(f"{name} of {t.dtype}; supported: {', '.join(str(x) for x in types)}")
    elif t.shape != like.shape or t.dtype != like.dtype or t.get_device() != like.get_device():
        _cuda(name, t, like)
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype}, got {tuple(t.shape)} {t.dtype}")
    return _ld(name, t)


def _out_shaped(name: str, out, shape, dtype, like: torch.Tensor) -> torch.Tensor:
    """The caller's output, checked, or a new one on `like`'s device."""
    if out is None:
        return like.new_empty(shape, dtype=dtype)
    _cuda(name, out, like)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError(f"{name} must be {tuple(shape)} {dtype}, got {tuple(out.shape)} {out.dtype}")
    return out


def _out(name: str, out, like: torch.Tensor, dtype) -> torch.Tensor:
    """The same with the shape of `like`; a new one is contiguous."""
    if out is None and like.is_contiguous():
        return torch.empty_like(like, dtype=dtype)       # the cheapest of torch's allocations
    return _out_shaped(name, out, like.shape, dtype, like)


def _span(t: torch.Tensor):
    """First byte and end of a tensor's storage range."""
    a = t.data_ptr()
    n = 1
    for size, stride in zip(t.shape, t.stride()):
        if size == 0:
            return a, a
        n += (size - 1) * stride
    return a, a + n * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors' elements may share memory: their storage ranges
    meet, and they are not different columns of rows with one stride."""
    a0, a1 = _span(a)
    b0, b1 = _span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if a.dim() == b.dim() == 2 and a.stride(1) == b.stride(1) == 1:
        es, ld = a.element_size(), a.stride(0)
        if ld and b.element_size() == es and b.stride(0) == ld and (b0 - a0) % es == 0:
            at = (b0 - a0) // es % ld                    # b's first column, seen from a's
            return not (at >= a.shape[1] and at + b.shape[1] <= ld)
    return True


def _apart(name: str, out: Optional[torch.Tensor], others, same=()) -> None:
    """A caller's output must not overlap `others`; it may be one of `same`
    itself (address, strides and type alike) but not overlap it otherwise."""
    if out is None:
        return
    if not isinstance(out, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(out).__name__}")
    for o in same:
        if o is None or (o.data_ptr() == out.data_ptr() and o.stride() == out.stride() and o.dtype == out.dtype):
            continue
        if _overlap(out, o):
            raise ValueError(f"{name} overlaps another operand")
    for o in others:
        if o is not None and _overlap(out, o):
            raise ValueError(f"{name} overlaps another operand")


# What the checks of a call's inputs found, by everything they look at: the
# inputs' types, shapes, strides and devices.  A program repeats few of them,
# and the checks cost more than a small call's launch.
_plans: dict = {}


def _look(call, *tensors):
    """The key of these inputs; None if one of them is not a tensor."""
    try:
        return (call, *[None if t is None else (t.dtype, t.shape, t.stride(), t.get_device()) for t in tensors])
    except (AttributeError, TypeError):
        return None


def _remember(key, plan):
    if key is not None:
        if len(_plans) >= 4096:
            _plans.clear()
        _plans[key] = plan
    return plan


def _norm_weight(weight, x, width: int) -> None:
    if not isinstance(weight, torch.Tensor) or weight.get_device() != x.get_device():
        _cuda("weight", weight, x)
    if weight.dim() != 1 or weight.shape[0] != width:
        raise ValueError(f"weight must be [{width}], got {tuple(weight.shape)}")
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise TypeError(f"weight must be {x.dtype} or torch.float32, got {weight.dtype}")
    _dense_last("weight", weight)
    if width < 1:
        raise ValueError("rows must have at least one element")


def _norm_plan(x, weight, residual):
    x_ld = _rows("x", x, types=_ROW_TYPES)
    rows, width = x.shape
    _norm_weight(weight, x, width)
    r_ld = 0 if residual is None else _rows("residual", residual, x)
    return x_ld, r_ld, rows, width, _DTYPE[x.dtype], _DTYPE[weight.dtype]


def _rms_norm(x, weight, residual, eps, out, scale_out, residual_out, stream, to8):
    key = _look("norm", x, weight, residual)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _norm_plan(x, weight, residual))
    x_ld, r_ld, rows, width, dt, wdt = plan
    eps = float(eps)
    given = [t for t in (out, scale_out, residual_out) if t is not None]
    if residual is None and residual_out is not None:
        raise ValueError("residual_out without residual")
    if out is not None:
        _apart("out", out, (residual, residual_out, weight, scale_out), (x,))
    if residual_out is not None:
        _apart("residual_out", residual_out, (weight, scale_out), (x, residual))
    if scale_out is not None:
        _apart("scale_out", scale_out, (x, residual, weight))
    _explicit(x, weight, residual, *given)
    raw, context = _on(x, stream, (x, weight, residual, out, scale_out, residual_out))
    with context:
        y_type = torch.float8_e4m3fn if to8 else x.dtype
        y = _out("out", out, x, y_type)
        scale = None
        if to8:
            scale = _out_shaped("scale_out", scale_out, (rows,), torch.float32, x)
            if scale_out is not None:
                _dense_last("scale_out", scale)
        h, h_ld = None, 0
        if residual is not None:
            h = _out("residual_out", residual_out, x, x.dtype)
            h_ld = width if residual_out is None else _ld("residual_out", h)
        rc = lib.bafe_cuda_rms_norm(
            x.data_ptr(), x_ld, None if residual is None else residual.data_ptr(), r_ld, weight.data_ptr(),
            y.data_ptr(), width if out is None else _ld("out", y), None if scale is None else scale.data_ptr(),
            None if h is None else h.data_ptr(), h_ld, rows, width, dt, wdt, DTYPE_E4M3 if to8 else dt, eps, raw)
        if rc:
            check(rc, "rms_norm")
    if given:
        _written(given)
    return y, scale, h


def rms_norm(x, weight, residual=None, *, eps: float = 1e-6, out=None, residual_out=None, stream=None):
    """Root-mean-square norm of each row of x [rows, width] (f32, f16, bf16):
    y = h / sqrt(mean(h^2) + eps) * weight with h = x, or h = x + residual
    rounded to x's type.  weight: [width] of x's type or f32.  Returns y, or
    (y, h) with a residual.  residual_out may be residual or x itself and
    out may be x itself; they must not overlap otherwise."""
    y, _, h = _rms_norm(x, weight, residual, eps, out, None, residual_out, stream, False)
    return y if h is None else (y, h)


def rms_norm_e4m3(x, weight, residual=None, *, eps: float = 1e-6, out=None, scale_out=None, residual_out=None,
                  stream=None):
    """rms_norm with 8-bit output: returns (q, scale) or (q, scale, h), where
    q [rows, width] (e4m3) times scale [rows] (f32) is the normed row;
    scale = max|y| / 448 of the row (1 for a row of zeros or with a NaN)."""
    q, scale, h = _rms_norm(x, weight, residual, eps, out, scale_out, residual_out, stream, True)
    return (q, scale) if h is None else (q, scale, h)


def _norm_grad_plan(dy, h, weight, dh):
    h_ld = _rows("h", h, types=_ROW_TYPES)
    dy_ld = _rows("dy", dy, h)
    dh_ld = 0 if dh is None else _rows("dh", dh, h)
    rows, width = h.shape
    _norm_weight(weight, h, width)
    with torch.cuda.device(h.get_device()):
        need = lib.bafe_cuda_rms_norm_grad_workspace(rows, width, _DTYPE[h.dtype])
    if need < 0:
        check(8, "rms_norm_grad")
    return h_ld, dy_ld, dh_ld, rows, width, _DTYPE[h.dtype], _DTYPE[weight.dtype], need


def rms_norm_grad(dy, h, weight, dh=None, *, eps: float = 1e-6, out=None, weight_out=None, stream=None):
    """Gradient of rms_norm: dy [rows, width] is y's gradient, h what was
    normed (rms_norm's second result, or x), dh the gradient that reaches h
    past the norm, if any.  Returns (dx, dweight): dx is the gradient of x
    and of the residual alike.  out may be dy or dh itself."""
    key = _look("norm_grad", dy, h, weight, dh)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _norm_grad_plan(dy, h, weight, dh))
    h_ld, dy_ld, dh_ld, rows, width, dt, wdt, need = plan
    eps = float(eps)
    if out is not None:
        _apart("out", out, (h, weight, weight_out), (dy, dh))
    if weight_out is not None:
        _apart("weight_out", weight_out, (dy, h, dh, weight))
    given = [t for t in (out, weight_out) if t is not None]
    _explicit(dy, h, weight, dh, *given)
    raw, context = _on(h, stream, (dy, h, weight, dh, out, weight_out))
    with context:
        dx = _out("out", out, h, h.dtype)
        dw = _out_shaped("weight_out", weight_out, (width,), weight.dtype, h)
        if weight_out is not None:
            _dense_last("weight_out", dw)
        ws = h.new_empty(need, dtype=torch.uint8)
        rc = lib.bafe_cuda_rms_norm_grad(
            dy.data_ptr(), dy_ld, h.data_ptr(), h_ld, weight.data_ptr(), None if dh is None else dh.data_ptr(), dh_ld,
            dx.data_ptr(), width if out is None else _ld("out", dx), dw.data_ptr(), rows, width, dt, wdt, eps,
            ws.data_ptr(), need, raw)
        if rc:
            check(rc, "rms_norm_grad")
    if given:
        _written(given)
    return dx, dw


def _scale_row(name: str, t, n: int, like: torch.Tensor) -> torch.Tensor:
    """Checks an f32 scale per row."""
    _cuda(name, t, like)
    if t.dim() != 1 or t.shape[0] != n or t.dtype != torch.float32:
        raise ValueError(f"{name} must be [{n}] torch.float32, got {tuple(t.shape)} {t.dtype}")
    _dense_last(name, t)
    return t


def _w4_plan(x, qweight, scales, zeros, x_scale, group):
    x_ld = _rows("x", x, types=(torch.float16, torch.bfloat16, torch.float8_e4m3fn))
    rows, k = x.shape
    to8 = x.dtype == torch.float8_e4m3fn
    if to8 != (x_scale is not None):
        raise ValueError("x_scale goes with e4m3 rows")
    if to8:
        _scale_row("x_scale", x_scale, rows, x)
    _cuda("qweight", qweight, x)
    if qweight.dim() != 2 or qweight.dtype != torch.uint8 or qweight.shape[1] != (k + 1) // 2:
        raise ValueError(f"qweight must be [n, {(k + 1) // 2}] torch.uint8, got {tuple(qweight.shape)} {qweight.dtype}")
    if group < 32 or group % 32:
        raise ValueError(f"group must be a positive multiple of 32, got {group}")
    if k < 1:
        raise ValueError("rows must have at least one element")
    n, groups = qweight.shape[0], -(-k // group)
    _cuda("scales", scales, x)
    if scales.shape != (n, groups):
        raise ValueError(f"scales must be [{n}, {groups}], got {tuple(scales.shape)}")
    if scales.dtype not in _ROW_TYPES:
        raise TypeError(f"scales must be f32, f16 or bf16, got {scales.dtype}")
    if zeros is not None:
        _cuda("zeros", zeros, x)
        if zeros.shape != (n, groups):
            raise ValueError(f"zeros must be [{n}, {groups}], got {tuple(zeros.shape)}")
        if zeros.dtype != torch.uint8:
            raise TypeError(f"zeros must be torch.uint8, got {zeros.dtype}")
    z_ld = 0 if zeros is None else _ld("zeros", zeros)
    dtype = x.dtype
    if to8:
        dtype = scales.dtype if scales.dtype in _HALF_TYPES else torch.bfloat16
    with torch.cuda.device(x.get_device()):
        need = lib.bafe_cuda_matvec_w4_workspace(rows, n, k, group)
    if need < 0:
        check(8, "matvec_w4")
    return x_ld, _ld("qweight", qweight), _ld("scales", scales), z_ld, rows, n, k, dtype, to8, need


def matvec_w4(x, qweight, scales, zeros=None, *, group: int = 128, x_scale=None, out=None, stream=None):
    """A few rows x [rows, k] times 4-bit weights [n, k]: returns [rows, n] of
        sum_g scales[n, g] * sum_{k in g} (q[n, k] - zeros[n, g]) * x[:, k].
    qweight: uint8 [n, ceil(k / 2)], byte j holding k = 2j in its low and
    2j + 1 in its high four bits; scales: [n, ceil(k / group)] f32, f16 or
    bf16; zeros: uint8 of the same shape (default 8); group: a
    multiple of 32.  x: f16, bf16, or e4m3 with x_scale, its f32 scale per row
    (as rms_norm_e4m3 returns them).  The result has x's type; for e4m3 the
    scales' 16-bit type, bf16 with f32 scales, or out's (f16 or bf16).
    The products (q - zeros) x are exact, sums in 32 bits; a row with an
    infinity or a NaN gives NaN throughout.  Meant for up to 32 rows; more read
    the weights again."""
    group = index(group)
    key = _look(("w4", group), x, qweight, scales, zeros, x_scale)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _w4_plan(x, qweight, scales, zeros, x_scale, group))
    x_ld, q_ld, s_ld, z_ld, rows, n, k, dtype, to8, need = plan
    y_ld = n
    if out is not None:
        _apart("out", out, (x, qweight, scales, zeros, x_scale))
        if to8:
            if out.dtype not in _HALF_TYPES:
                raise TypeError(f"out must be f16 or bf16, got {out.dtype}")
            dtype = out.dtype
        _out_shaped("out", out, (rows, n), dtype, x)
        y_ld = _ld("out", out)
    _explicit(x, scales, x_scale, out)
    raw, context = _on(x, stream, (x, qweight, scales, zeros, x_scale, out))
    with context:
        y = out if out is not None else x.new_empty((rows, n), dtype=dtype)
        ws = x.new_empty(need, dtype=torch.uint8) if need else None
        rc = lib.bafe_cuda_matvec_w4(
            x.data_ptr(), x_ld, None if x_scale is None else x_scale.data_ptr(), qweight.data_ptr(), q_ld,
            scales.data_ptr(), s_ld, None if zeros is None else zeros.data_ptr(), z_ld, y.data_ptr(), y_ld, rows, n, k,
            group, _DTYPE[x.dtype], _DTYPE[scales.dtype], _DTYPE[dtype], None if ws is None else ws.data_ptr(), need,
            raw)
        if rc:
            check(rc, "matvec_w4")
    if out is not None:
        _written((out,))
    return y


def _offsets(offsets, x, experts: Optional[int] = None) -> int:
    """Checks the experts' row offsets; their number of experts."""
    _cuda("offsets", offsets, x)
    if offsets.dim() != 1 or offsets.dtype != torch.int32 or offsets.shape[0] < 2:
        raise ValueError(f"offsets must be [experts + 1] torch.int32, got {tuple(offsets.shape)} {offsets.dtype}")
    _dense_last("offsets", offsets)
    if experts is not None and offsets.shape[0] != experts + 1:
        raise ValueError(f"offsets must have {experts + 1} entries for {experts} experts, got {offsets.shape[0]}")
    return offsets.shape[0] - 1


def _workspace(need: int, what: str, like: torch.Tensor):
    if need < 0:
        check(8, what)
    return like.new_empty(need, dtype=torch.uint8) if need else None


def _grouped_plan(x, w, offsets, x_scale, w_scale, transposed):
    """transposed: w's two last dimensions are exchanged (the gradient of the rows)."""
    name = "dy" if transposed else "x"
    x_ld = _rows(name, x, types=_HALF_TYPES if transposed else (torch.float16, torch.bfloat16, torch.float8_e4m3fn))
    _cuda("w", w, x)
    if w.dim() != 3:
        raise ValueError(f"w must be [experts, n, k], got {tuple(w.shape)}")
    if transposed:
        w = w.transpose(1, 2)
    to8 = x.dtype == torch.float8_e4m3fn
    rows = x.shape[0]
    experts, n, k = w.shape
    if x.shape[1] != k:
        raise ValueError(f"{name} has rows of {x.shape[1]} elements for weights of {k}")
    if w.dtype != x.dtype:
        raise TypeError(f"weights of {w.dtype} for rows of {x.dtype}")
    if min(experts, n, k) < 1:
        raise ValueError(f"empty weights {tuple(w.shape)}")
    _offsets(offsets, x, experts)
    # contiguous along k (as made), or along n (the transposed storage)
    if k == 1 or w.stride(2) == 1:
        kmajor, ld, inner = 1, (w.stride(1) if n > 1 else k), k
    elif n == 1 or w.stride(1) == 1:
        kmajor, ld, inner = 0, (w.stride(2) if k > 1 else n), n
    else:
        raise ValueError("one of the weights' two last dimensions must be contiguous")
    outer = n if kmajor else k
    stride = w.stride(0) if experts > 1 else outer * ld
    if ld < inner or (experts > 1 and stride < (outer - 1) * ld + inner):
        raise ValueError("the experts' weights overlap")
    s_ld = 0
    if to8:
        if not kmajor:
            raise ValueError("e4m3 weights must be contiguous along k")
        if x_scale is None or w_scale is None:
            raise ValueError("e4m3 operands take x_scale and w_scale")
        _scale_row("x_scale", x_scale, rows, x)
        _cuda("w_scale", w_scale, x)
        if w_scale.shape != (experts, n) or w_scale.dtype != torch.float32:
            raise ValueError(f"w_scale must be [{experts}, {n}] torch.float32, "
                             f"got {tuple(w_scale.shape)} {w_scale.dtype}")
        s_ld = _ld("w_scale", w_scale)
    elif x_scale is not None or w_scale is not None:
        raise ValueError("scales go with e4m3 operands")
    return x_ld, ld, stride, kmajor, s_ld, rows, experts, n, k, _DTYPE[x.dtype], to8


def _grouped(what, x, w, offsets, x_scale, w_scale, out, stream, transposed):
    key = _look(what, x, w, offsets, x_scale, w_scale)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _grouped_plan(x, w, offsets, x_scale, w_scale, transposed))
    x_ld, w_ld, stride, kmajor, s_ld, rows, experts, n, k, dt, to8 = plan
    dtype, y_ld = torch.bfloat16 if to8 else x.dtype, n
    if out is not None:
        _apart("out", out, (x, w, offsets, x_scale, w_scale))
        if to8:
            if out.dtype not in _HALF_TYPES:
                raise TypeError(f"out must be f16 or bf16, got {out.dtype}")
            dtype = out.dtype
        _out_shaped("out", out, (rows, n), dtype, x)
        y_ld = _ld("out", out)
    _explicit(x, w, x_scale, w_scale, out)
    raw, context = _on(x, stream, (x, w, offsets, x_scale, w_scale, out))
    with context:
        y = out if out is not None else x.new_empty((rows, n), dtype=dtype)
        xp, wp = x.data_ptr(), w.data_ptr()
        ws, need = None, 0
        if (xp | wp | (x_ld | w_ld | stride) * x.element_size()) & 15:      # rows off 16-byte boundaries
            need = lib.bafe_cuda_grouped_matmul_workspace(xp, x_ld, wp, w_ld, stride, kmajor, rows, experts, n, k, dt)
            ws = _workspace(need, what, x)
        rc = lib.bafe_cuda_grouped_matmul(
            xp, x_ld, wp, w_ld, stride, kmajor, offsets.data_ptr(), None if x_scale is None else x_scale.data_ptr(),
            None if w_scale is None else w_scale.data_ptr(), s_ld, y.data_ptr(), y_ld, rows, experts, n, k, dt,
            _DTYPE[dtype], None if ws is None else ws.data_ptr(), need, raw)
        if rc:
            check(rc, what)
    if out is not None:
        _written((out,))
    return y


def grouped_matmul(x, w, offsets, *, x_scale=None, w_scale=None, out=None, stream=None):
    """Products grouped by expert: rows offsets[e] .. offsets[e + 1] of x
    [rows, k], sorted by expert, times w[e].T; w: [experts, n, k], contiguous
    along k or along n; offsets: int32 [experts + 1] on the device, ascending
    (clamped to [0, rows]); experts may have no rows.  f16 or bf16, the result
    [rows, n] alike; or both e4m3 (w contiguous along k) with x_scale [rows]
    and w_scale [experts, n], f32, which multiply the sums: the result is bf16
    or out's type (f16, bf16).  Rows before the first and behind the last
    group are left as they are in out (unset in a fresh result).  No host
    synchronisation."""
    return _grouped("grouped_matmul", x, w, offsets, x_scale, w_scale, out, stream, False)


def grouped_matmul_grad_input(dy, w, offsets, *, out=None, stream=None):
    """Gradient of grouped_matmul's x: dy [rows, n] times w[e] for each
    expert's rows -> [rows, k].  f16 or bf16; w as in the forward call."""
    return _grouped("grouped_matmul_grad_input", dy, w, offsets, None, None, out, stream, True)


def _grad_weight_plan(dy, x, offsets):
    dy_ld = _rows("dy", dy, types=_HALF_TYPES)
    x_ld = _rows("x", x, types=_HALF_TYPES)
    if x.get_device() != dy.get_device() or x.dtype != dy.dtype or x.shape[0] != dy.shape[0]:
        raise ValueError(f"dy {tuple(dy.shape)} {dy.dtype} and x {tuple(x.shape)} {x.dtype} do not belong together")
    experts = _offsets(offsets, dy)
    rows, n, k = dy.shape[0], dy.shape[1], x.shape[1]
    if min(n, k) < 1:
        raise ValueError("rows must have at least one element")
    return dy_ld, x_ld, experts, rows, n, k, _DTYPE[dy.dtype]


def grouped_matmul_grad_weight(dy, x, offsets, *, out=None, stream=None):
    """Gradient of grouped_matmul's w: dw[e] = dy_e.T @ x_e over expert e's
    rows, [experts, n, k]; zeros for an expert without rows.  dy [rows, n]
    and x [rows, k], both f16 or both bf16.  Rows outside all groups do not
    count, whatever they hold."""
    key = _look("grad_weight", dy, x, offsets)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _grad_weight_plan(dy, x, offsets))
    dy_ld, x_ld, experts, rows, n, k, dt = plan
    ld, stride = k, n * k
    if out is not None:
        _apart("out", out, (dy, x, offsets))
        _out_shaped("out", out, (experts, n, k), dy.dtype, dy)
        _dense_last("out", out)
        ld = out.stride(1) if n > 1 else k
        stride = out.stride(0) if experts > 1 else n * ld
        if ld < k or stride < (n - 1) * ld + k:
            raise ValueError("out's rows overlap")
    _explicit(dy, x, out)
    raw, context = _on(dy, stream, (dy, x, offsets, out))
    with context:
        dw = out if out is not None else dy.new_empty((experts, n, k))
        dyp, xp = dy.data_ptr(), x.data_ptr()
        ws, need = None, 0
        if (dyp | xp | (dy_ld | x_ld) * 2) & 15:         # rows off 16-byte boundaries
            need = lib.bafe_cuda_grouped_matmul_grad_weight_workspace(dyp, dy_ld, xp, x_ld, rows, n, k)
            ws = _workspace(need, "grouped_matmul_grad_weight", dy)
        rc = lib.bafe_cuda_grouped_matmul_grad_weight(
            dyp, dy_ld, xp, x_ld, offsets.data_ptr(), dw.data_ptr(), ld, stride, rows, experts, n, k, dt,
            None if ws is None else ws.data_ptr(), need, raw)
        if rc:
            check(rc, "grouped_matmul_grad_weight")
    if out is not None:
        _written((out,))
    return dw


# A contiguous tensor on the current device, by the shortest way that torch has (0.9 us
# against 2.1 for new_empty with a type); the calls below allocate with their tensors'
# device current.  It passes by dispatch modes and does not fill fresh memory where torch is
# asked to be deterministic: there, and where it is missing, the public way is taken.
_strided = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)
_modes = getattr(torch._C, "_len_torch_dispatch_stack", None)
_deterministic = torch._C._get_deterministic_algorithms  # what torch.are_deterministic_algorithms_enabled reads
if _modes is None:
    _strided = None


def _new(shape, dtype) -> torch.Tensor:
    if _strided is None or _modes() or _deterministic():
        return torch.empty(shape, dtype=dtype, device="cuda")
    return _strided(shape, (1,) if len(shape) == 1 else (shape[1], 1), dtype)


class Routing(NamedTuple):
    """What route returns; offsets and place are as grouped_matmul, dispatch and combine take them."""
    weights: torch.Tensor
    experts: torch.Tensor
    offsets: torch.Tensor
    place: torch.Tensor


_SCORE = {"softmax": 0, "sigmoid": 1}


def _score(score) -> int:
    code = _SCORE.get(score) if isinstance(score, str) else None
    if code is None:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    return code


def _route_plan(logits, bias, k):
    ld = _rows("logits", logits, types=_ROW_TYPES)
    rows, experts = logits.shape
    if not 1 <= experts <= 1024:
        raise ValueError(f"logits must have 1 to 1024 columns, got {experts}")
    if not 1 <= k <= min(experts, 31):
        raise ValueError(f"k must be between 1 and {min(experts, 31)}, got {k}")
    if bias is not None:
        _cuda("bias", bias, logits)
        if bias.dim() != 1 or bias.shape[0] != experts or bias.dtype != torch.float32:
            raise ValueError(f"bias must be [{experts}] torch.float32, got {tuple(bias.shape)} {bias.dtype}")
        _dense_last("bias", bias)
    with torch.cuda.device(logits.get_device()):
        need = lib.bafe_cuda_route_workspace(rows, experts, k)
    if need < 0:
        check(8, "route")
    return ld, rows, experts, _DTYPE[logits.dtype], need


def route(logits, k: int, *, score: str = "softmax", bias=None, groups: int = 1, keep_groups: int = 1,
          group_top: int = 2, renormalize: bool = True, scale: float = 1.0, stream=None) -> Routing:
    """Chooses k experts for each row of a router's logits [rows, experts]
    (f32, f16, bf16) and lays the rows out by expert.  With s = softmax or
    sigmoid of the logits and c = s + bias (f32 [experts]; it counts for the
    choice only):
      * groups > 1: of so many groups of consecutive experts the keep_groups
        best stay, by the sum of their group_top (1 or 2) largest c;
      * experts [rows, k] (int32): those of the k largest c, best first, the
        lower index of equals: with a bias by c in 64 bits, where scores below
        e^-700 count as 0, as they do in the groups' worths; without one by the
        logits, whose order goes on where scores are equal (sigmoids of 38 and 40);
      * weights [rows, k] (f32): s of them, with renormalize over their sum,
        times scale.
    An expert whose logit is -inf is shut: never chosen, and without a chosen
    one left the expert is -1 and the weight 0, so that a row of -inf
    (padding) goes nowhere.  A row with a NaN (softmax: or a +inf) gets
    experts 0 .. k - 1 and NaN weights.
    offsets [experts + 1] and place [rows, k] (int32): choice j of row t is row
    place[t, j] of the choices sorted by expert (-1: none), expert e's are
    offsets[e] .. offsets[e + 1].  k <= 31, experts <= 1024, groups <= 32."""
    code, k, groups, keep_groups, group_top = _score(score), index(k), index(groups), index(keep_groups), index(group_top)
    key = _look(("route", k), logits, bias)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _route_plan(logits, bias, k))
    ld, rows, experts, dt, need = plan
    if groups == 1 and keep_groups != 1 or not 1 <= groups <= 32 or experts % groups:
        raise ValueError(f"{groups} groups, {keep_groups} kept, of {experts} experts: "
                         "groups must be a divisor of at most 32, of which some stay")
    if not 1 <= keep_groups <= groups or experts // groups * keep_groups < k:
        raise ValueError(f"{keep_groups} groups of {experts // groups} experts must be at most {groups} and hold k = {k}")
    if group_top not in (1, 2):
        raise ValueError(f"group_top must be 1 or 2, got {group_top}")
    _explicit(logits, bias)
    raw, context = _on(logits, stream, (logits, bias))
    with context:
        weights = _new((rows, k), torch.float32)
        chosen = _new((rows, k), torch.int32)
        place = _new((rows, k), torch.int32)
        offsets = _new((experts + 1,), torch.int32)
        ws = _new((need,), torch.uint8) if need else None
        rc = lib.bafe_cuda_route(
            logits.data_ptr(), ld, None if bias is None else bias.data_ptr(), weights.data_ptr(), chosen.data_ptr(),
            offsets.data_ptr(), place.data_ptr(), rows, experts, k, groups, keep_groups, group_top, code,
            bool(renormalize), float(scale), dt, None if ws is None else ws.data_ptr(), need, raw)
        if rc:
            check(rc, "route")
    return Routing(weights, chosen, offsets, place)


def _choices(name: str, t, rows: int, like: torch.Tensor, dtype, k: Optional[int] = None) -> int:
    """Checks a [rows, k] tensor of the choices; its row stride (0: one row for all)."""
    _cuda(name, t, like)
    if t.dim() != 2 or t.shape[0] != rows or t.dtype != dtype or (k is not None and t.shape[1] != k):
        raise ValueError(f"{name} must be [{rows}, {'k' if k is None else k}] {dtype}, got {tuple(t.shape)} {t.dtype}")
    if not 1 <= t.shape[1] <= 31:
        raise ValueError(f"{name} must have 1 to 31 columns, got {t.shape[1]}")
    _dense_last(name, t)
    return t.stride(0) if rows > 1 else t.shape[1]


def _own_rows(name: str, ld: int, k: int) -> int:
    if ld < k:
        raise ValueError(f"{name}'s rows overlap")
    return ld


def _route_grad_plan(dweights, logits, experts):
    ld = _rows("logits", logits, types=_ROW_TYPES)
    rows, n = logits.shape
    if not 1 <= n <= 1024:
        raise ValueError(f"logits must have 1 to 1024 columns, got {n}")
    e_ld = _choices("experts", experts, rows, logits, torch.int32)
    k = experts.shape[1]
    if k > n:
        raise ValueError(f"{k} choices of {n} experts")
    d_ld = _choices("dweights", dweights, rows, logits, torch.float32, k)
    return ld, _own_rows("experts", e_ld, k), d_ld, rows, n, k, _DTYPE[logits.dtype]


def route_grad(dweights, logits, experts, *, score: str = "softmax", renormalize: bool = True, scale: float = 1.0,
               out=None, stream=None):
    """Gradient of route's weights: dweights [rows, k] (f32), logits and the
    chosen experts as route took and returned them -> [rows, experts] of the
    logits' type.  score, renormalize and scale as in the forward call; the
    choice itself and the bias have no gradient.  Experts outside 0 ..
    experts - 1 (-1: none) count for nothing; a row names no expert twice.
    out may be logits itself."""
    code = _score(score)
    key = _look("route_grad", dweights, logits, experts)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _route_grad_plan(dweights, logits, experts))
    ld, e_ld, d_ld, rows, n, k, dt = plan
    if out is not None:
        _apart("out", out, (dweights, experts), (logits,))
    _explicit(dweights, logits, out)
    raw, context = _on(logits, stream, (dweights, logits, experts, out))
    with context:
        dlogits = _new((rows, n), logits.dtype) if out is None else _out("out", out, logits, logits.dtype)
        rc = lib.bafe_cuda_route_grad(
            dweights.data_ptr(), d_ld, logits.data_ptr(), ld, experts.data_ptr(), e_ld, dlogits.data_ptr(),
            n if out is None else _ld("out", dlogits), rows, n, k, code, bool(renormalize), float(scale), dt, raw)
        if rc:
            check(rc, "route_grad")
    if out is not None:
        _written((out,))
    return dlogits


def _dispatch_plan(x, place, scale):
    x_ld = _rows("x", x, types=tuple(_DTYPE))
    rows, width = x.shape
    if width < 1:
        raise ValueError("rows must have at least one element")
    p_ld = _choices("place", place, rows, x, torch.int32)
    k = place.shape[1]
    if scale is not None:
        _scale_row("scale", scale, rows, x)
    return x_ld, _own_rows("place", p_ld, k), rows, width, k


def dispatch(x, place, *, scale=None, out=None, scale_out=None, stream=None):
    """Rows laid out by expert: y[place[t, j]] = x[t].  x: [rows, width] (f32,
    f16, bf16, e4m3); place: int32 [rows, k] as route returns it, no row of y
    twice (others than 0 .. n - 1 count for nothing).  y has rows * k rows, or is
    out [n, width]; rows that no place names are left as they are in out
    (unset in a fresh result).  With scale (f32 [rows], as rms_norm_e4m3
    returns it) returns (y, its scale [n]).  The gradient is combine(dy,
    place)."""
    key = _look("dispatch", x, place, scale)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _dispatch_plan(x, place, scale))
    x_ld, p_ld, rows, width, k = plan
    if scale is None and scale_out is not None:
        raise ValueError("scale_out without scale")
    n, y_ld = rows * k, width
    given = [t for t in (out, scale_out) if t is not None]
    if out is not None:
        _apart("out", out, (x, place, scale, scale_out))
        if out.dim() != 2:
            raise ValueError(f"out must have two dimensions, got {tuple(out.shape)}")
        n = out.shape[0]
        _out_shaped("out", out, (n, width), x.dtype, x)
        y_ld = _ld("out", out)
    if scale_out is not None:
        _apart("scale_out", scale_out, (x, place, scale))
        _scale_row("scale_out", scale_out, n, x)
    _explicit(x, scale, *given)
    raw, context = _on(x, stream, (x, place, scale, out, scale_out))
    with context:
        y = out if out is not None else _new((n, width), x.dtype)
        s = scale_out
        if scale is not None and s is None:
            s = _new((n,), torch.float32)
        rc = lib.bafe_cuda_dispatch(
            x.data_ptr(), x_ld, None if scale is None else scale.data_ptr(), place.data_ptr(), p_ld, y.data_ptr(), y_ld,
            None if s is None else s.data_ptr(), rows, k, n, width, x.element_size(), raw)
        if rc:
            check(rc, "dispatch")
    if given:
        _written(given)
    return y if scale is None else (y, s)


def _combine_plan(y, place, weights):
    y_ld = _rows("y", y, types=_ROW_TYPES)
    n, width = y.shape
    if width < 1:
        raise ValueError("rows must have at least one element")
    _cuda("place", place, y)
    rows = place.shape[0] if place.dim() else 0
    p_ld = _choices("place", place, rows, y, torch.int32)
    k = place.shape[1]
    w_ld = 0 if weights is None else _choices("weights", weights, rows, y, torch.float32, k)
    return y_ld, _own_rows("place", p_ld, k), w_ld, rows, k, n, width, _DTYPE[y.dtype]


def combine(y, place, weights=None, *, out=None, stream=None):
    """The experts' rows summed for each token: [rows, width] of
        out[t] = sum_j weights[t, j] * y[place[t, j]].
    y: [n, width] (f32, f16, bf16); place: int32 [rows, k], others than 0 ..
    n - 1 (-1: none) count for nothing; weights: f32 [rows, k] (default 1).
    Summed in 32 bits in the order of j, rounded once.  Without weights and
    with y's gradient for y it is the gradient of dispatch."""
    key = _look("combine", y, place, weights)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _combine_plan(y, place, weights))
    y_ld, p_ld, w_ld, rows, k, n, width, dt = plan
    out_ld = width
    if out is not None:
        _apart("out", out, (y, place, weights))
        _out_shaped("out", out, (rows, width), y.dtype, y)
        out_ld = _ld("out", out)
    _explicit(y, weights, out)
    raw, context = _on(y, stream, (y, place, weights, out))
    with context:
        r = out if out is not None else _new((rows, width), y.dtype)
        rc = lib.bafe_cuda_combine(
            y.data_ptr(), y_ld, place.data_ptr(), p_ld, None if weights is None else weights.data_ptr(), w_ld,
            r.data_ptr(), out_ld, rows, k, n, width, dt, raw)
        if rc:
            check(rc, "combine")
    if out is not None:
        _written((out,))
    return r


def _combine_grad_plan(dout, y, place, weights):
    plan = _combine_plan(y, place, weights)
    rows, width = plan[3], plan[6]
    _cuda("dout", dout, y)
    if tuple(dout.shape) != (rows, width) or dout.dtype != y.dtype:
        raise ValueError(f"dout must be {(rows, width)} {y.dtype}, got {tuple(dout.shape)} {dout.dtype}")
    _dense_last("dout", dout)
    return (dout.stride(0) if rows > 1 else width,) + plan


def combine_grad(dout, y, place, weights, *, out=None, weight_out=None, stream=None):
    """Gradient of combine with weights: (dy [n, width], dweights [rows, k]
    f32) with
        dy[place[t, j]] = weights[t, j] * dout[t],
        dweights[t, j] = sum(dout[t] * y[place[t, j]])   (0 without a place).
    place names no row of y twice; rows that it does not name are left as they
    are in out (unset in a fresh result).  out may be y itself.  (Without
    weights, dispatch(dout, place) is the gradient.)"""
    if weights is None:
        raise ValueError("combine_grad takes weights; without them the gradient is dispatch(dout, place)")
    key = _look("combine_grad", dout, y, place, weights)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _combine_grad_plan(dout, y, place, weights))
    d_ld, y_ld, p_ld, w_ld, rows, k, n, width, dt = plan
    given = [t for t in (out, weight_out) if t is not None]
    out_ld = width
    if out is not None:
        _apart("out", out, (dout, place, weights, weight_out), (y,))
        _out_shaped("out", out, (n, width), y.dtype, y)
        out_ld = _ld("out", out)
    if weight_out is not None:
        _apart("weight_out", weight_out, (dout, y, place, weights))
        _out_shaped("weight_out", weight_out, (rows, k), torch.float32, y)
        if not weight_out.is_contiguous():
            raise ValueError("weight_out must be contiguous")
    _explicit(dout, y, weights, *given)
    raw, context = _on(y, stream, (dout, y, place, weights, out, weight_out))
    with context:
        dy = out if out is not None else _new((n, width), y.dtype)
        dw = weight_out if weight_out is not None else _new((rows, k), torch.float32)
        rc = lib.bafe_cuda_combine_grad(
            dout.data_ptr(), d_ld, y.data_ptr(), y_ld, place.data_ptr(), p_ld, weights.data_ptr(), w_ld, dy.data_ptr(),
            out_ld, dw.data_ptr(), rows, k, n, width, dt, raw)
        if rc:
            check(rc, "combine_grad")
    if given:
        _written(given)
    return dy, dw


def _loss_plan(x, w, target, gradient):
    x_ld = _rows("x", x, types=_HALF_TYPES)
    w_ld = _rows("w", w, types=_HALF_TYPES)
    if w.dtype != x.dtype or w.get_device() != x.get_device() or w.shape[1] != x.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} {x.dtype} and w {tuple(w.shape)} {w.dtype} do not belong together")
    rows, width = x.shape
    vocab = w.shape[0]
    if min(vocab, width) < 1:
        raise ValueError(f"empty weights {tuple(w.shape)}")
    _cuda("target", target, x)
    if target.dim() != 1 or target.shape[0] != rows or target.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"target must be [{rows}] torch.int64 or torch.int32, got {tuple(target.shape)} {target.dtype}")
    _dense_last("target", target)
    with torch.cuda.device(x.get_device()):
        need = lib.bafe_cuda_linear_cross_entropy_workspace(None, x_ld, None, w_ld, rows, vocab, width, gradient)
    if need < 0:
        check(8, "linear_cross_entropy")
    return x_ld, w_ld, rows, vocab, width, target.element_size(), _DTYPE[x.dtype], need


def _int64(name: str, value) -> int:
    value = index(value)
    if not -(1 << 63) <= value < 1 << 63:
        raise ValueError(f"{name} must fit into 64 bits, got {value}")
    return value


def _loss_workspace(x, x_ld, w, w_ld, rows, vocab, width, gradient, need):
    """Scratch of a call: more than planned where an operand starts off a 16-byte boundary."""
    xp, wp = x.data_ptr(), w.data_ptr()
    if (xp | wp) & 15:
        need = lib.bafe_cuda_linear_cross_entropy_workspace(xp, x_ld, wp, w_ld, rows, vocab, width, gradient)
    if need < 0:
        check(8, "linear_cross_entropy")
    return (_new((need,), torch.uint8) if need else None), need


def linear_cross_entropy(x, w, target, *, ignore_index: int = -100, stream=None):
    """Softmax cross entropy of the logits z = x @ w.T, which are not kept: x
    [rows, width] hidden states, w [vocab, width] output weights (both f16 or
    both bf16), target [rows] (int64 or int32).  Returns (loss, lse), f32 [rows]:
        lse = log(sum(exp(z))),  loss = lse - z[target],
    loss 0 where target is ignore_index and NaN where it is out of range
    otherwise.  Logits are summed and used in 32 bits.  Keep lse for the gradient.
    Scratch: 16 bytes for every row and 256 words, up to 128 MB and 20 bytes a
    row (1 MB up to 128 rows), and a copy of x or w whose rows start off 16-byte
    boundaries."""
    key = _look("loss", x, w, target)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _loss_plan(x, w, target, 0))
    x_ld, w_ld, rows, vocab, width, tb, dt, need = plan
    ignore_index = _int64("ignore_index", ignore_index)
    _explicit(x, w)
    raw, context = _on(x, stream, (x, w, target))
    with context:
        loss = _new((rows,), torch.float32)
        lse = _new((rows,), torch.float32)
        ws, need = _loss_workspace(x, x_ld, w, w_ld, rows, vocab, width, 0, need)
        rc = lib.bafe_cuda_linear_cross_entropy(
            x.data_ptr(), x_ld, w.data_ptr(), w_ld, target.data_ptr(), tb, loss.data_ptr(), lse.data_ptr(), rows, vocab,
            width, ignore_index, dt, None if ws is None else ws.data_ptr(), need, raw)
        if rc:
            check(rc, "linear_cross_entropy")
    return loss, lse


def _loss_grad_plan(dloss, x, w, target, lse):
    plan = _loss_plan(x, w, target, 1)
    rows = plan[2]
    _cuda("dloss", dloss, x)
    if dloss.dim() != 1 or dloss.shape[0] != rows or dloss.dtype != torch.float32:
        raise ValueError(f"dloss must be [{rows}] torch.float32, got {tuple(dloss.shape)} {dloss.dtype}")
    _scale_row("lse", lse, rows, x)
    return (dloss.stride(0) if rows > 1 else 1,) + plan


def linear_cross_entropy_grad(dloss, x, w, target, lse, *, ignore_index: int = -100, out=None, weight_out=None,
                              stream=None):
    """Gradient of linear_cross_entropy: (dx [rows, width], dw [vocab, width])
    of x's type, from dloss [rows] (f32, any stride: an expanded one value
    too) and the forward call's arguments and lse:
        g = dloss * (exp(z - lse) - onehot(target)),  dx = g @ w,  dw = g.T @ x.
    Rows whose target is ignore_index add nothing (their x has to be finite all
    the same); one out of range gives NaN.  g is rounded to x's type (in f16 an
    entry is off by 2^-40 of the largest counted dloss at least, so rows far
    below that, by 2^-20 or more, have fewer bits), sums are in 32 bits.  out and
    weight_out must not overlap any operand.
    Scratch: g for a piece of the vocabulary at a time (up to 512 MB, beyond
    65536 rows 8 KB a row); dx's sums in 32 bits where there is more than one
    piece, or few rows and columns share a long one (4 bytes an element, in the
    second case up to 1 GB of them); a copy of x or w as above."""
    key = _look("loss_grad", dloss, x, w, target, lse)
    plan = _plans.get(key)
    if plan is None:
        plan = _remember(key, _loss_grad_plan(dloss, x, w, target, lse))
    d_ld, x_ld, w_ld, rows, vocab, width, tb, dt, need = plan
    ignore_index = _int64("ignore_index", ignore_index)
    given = [t for t in (out, weight_out) if t is not None]
    dx_ld = dw_ld = width
    if out is not None:
        _apart("out", out, (dloss, x, w, target, lse, weight_out))
        _out_shaped("out", out, (rows, width), x.dtype, x)
        dx_ld = _ld("out", out)
    if weight_out is not None:
        _apart("weight_out", weight_out, (dloss, x, w, target, lse))
        _out_shaped("weight_out", weight_out, (vocab, width), x.dtype, x)
        dw_ld = _ld("weight_out", weight_out)
    _explicit(dloss, x, w, lse, *given)
    raw, context = _on(x, stream, (dloss, x, w, target, lse, out, weight_out))
    with context:
        dx = out if out is not None else _new((rows, width), x.dtype)
        dw = weight_out if weight_out is not None else _new((vocab, width), x.dtype)
        ws, need = _loss_workspace(x, x_ld, w, w_ld, rows, vocab, width, 1, need)
        rc = lib.bafe_cuda_linear_cross_entropy_grad(
            dloss.data_ptr(), d_ld, x.data_ptr(), x_ld, w.data_ptr(), w_ld, target.data_ptr(), tb, lse.data_ptr(),
            dx.data_ptr(), dx_ld, dw.data_ptr(), dw_ld, rows, vocab, width, ignore_index, dt,
            None if ws is None else ws.data_ptr(), need, raw)
        if rc:
            check(rc, "linear_cross_entropy_grad")
    if given:
        _written(given)
    return dx, dw


__all__ = ["rms_norm", "rms_norm_e4m3", "rms_norm_grad", "grouped_matmul", "grouped_matmul_grad_input",
           "grouped_matmul_grad_weight", "matvec_w4", "Routing", "route", "route_grad", "dispatch", "combine",
           "combine_grad", "linear_cross_entropy", "linear_cross_entropy_grad"]
