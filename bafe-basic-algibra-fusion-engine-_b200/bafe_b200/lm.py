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
from typing import Optional

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


__all__ = ["rms_norm", "rms_norm_e4m3", "rms_norm_grad", "grouped_matmul", "grouped_matmul_grad_input",
           "grouped_matmul_grad_weight", "matvec_w4"]
