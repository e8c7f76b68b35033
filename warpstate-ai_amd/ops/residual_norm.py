"""Residual addition and RMSNorm in one pass on gfx950, in BF16 with autograd or in 8 bits.

Between two projections of a layer the first one's output is added to the residual stream and the
sum is normalized for the second (warpstate/model.py:174-178; separate operators there and in
``activation_execution.bf16_rmsnorm``). With s the new stream,

    s = r(x + residual),   y = s rstd w,   rstd = 1 / sqrt(mean(s^2) + eps)

* ``add_rmsnorm``: (y, s) with autograd to x, the residual and the weight. y is rounded once, to
  BF16 (``bf16_rmsnorm`` rounds s rstd first, as the reference's eager module does).
* ``rmsnorm_quantize``: y as the e4m3 operand of ``fp8_execution.fp8_mm``, quantized from FP32,
  for inference.

The stream is BF16 or FP32 and keeps its type. First derivatives by reverse mode only:
forward-mode tensors and functorch's derivatives are refused, and so is a second
differentiation.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from ops import _hip
from ops.fp8_execution import _SCALE_TYPES, E8M0, _blocks, _data, _scales, _views

BF16, F32 = torch.bfloat16, torch.float32
MAX_WIDTH = 8192
Tensor = torch.Tensor


def _rows(t: Tensor) -> Tensor:
    """t's rows of its last dimension, with a unit column stride and no overlap: a view or a
    copy."""
    cols = t.shape[-1]
    t = t.reshape(t.numel() // cols, cols)
    if (t.stride(1) == 1 or cols == 1) and (t.shape[0] <= 1 or t.stride(0) >= cols):
        return t
    return t.contiguous()


def _row_stride(t: Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check(x: Tensor, residual: Tensor | None, weight: Tensor) -> None:
    if x.dtype != BF16 or x.ndim < 1:
        raise ValueError("Expected BF16 rows")
    d = x.shape[-1]
    if not 1 <= d <= MAX_WIDTH:
        raise ValueError(f"RMSNorm takes rows of 1 to {MAX_WIDTH} columns, not {d}")
    if weight.dtype != F32 or weight.shape != (d,) or weight.device != x.device:
        raise ValueError(f"The norm's weight must be a vector of {d} values on {x.device}")
    if residual is not None and (residual.dtype not in (BF16, F32) or residual.shape != x.shape
                                 or residual.device != x.device):
        raise ValueError(f"The residual must be BF16 or FP32, of shape {list(x.shape)} on "
                         f"{x.device}")


def _refuse_tangents(name: str, *tensors: Tensor | None) -> None:
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


class _Once(torch.autograd.Function):
    """The first ``count`` tensors, behind a node that depends on all of them and refuses to be
    differentiated."""

    @staticmethod
    def forward(ctx, message, count, *tensors):
        ctx.message = message
        return tuple(t.view_as(t) for t in tensors[:count])

    @staticmethod
    def backward(ctx, *_grads):
        raise RuntimeError(ctx.message)


def _once(name: str, grads: tuple, *sources: Tensor | None) -> tuple:
    """``grads`` (tensors and None) of a backward; where a graph of it is recorded, they depend on
    ``sources`` and refuse a second derivative."""
    sources = [t for t in sources if t is not None and t.requires_grad]
    if not torch.is_grad_enabled() or not sources:
        return grads
    known = [g for g in grads if g is not None]
    wrapped = iter(_Once.apply(f"{name} cannot be differentiated twice", len(known), *known,
                               *sources))
    return tuple(None if g is None else next(wrapped) for g in grads)


class _AddRmsnorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        a, r, w = _rows(x), _rows(residual), weight.contiguous()
        rows, d = a.shape
        y = torch.empty(x.shape, dtype=BF16, device=x.device)
        stream = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
        _hip.call_on(x, "ws_add_rmsnorm", a.data_ptr(), _row_stride(a), r.data_ptr(),
                     _row_stride(r), int(r.dtype == F32), w.data_ptr(), eps, rows, d, y.data_ptr(),
                     stream.data_ptr())
        ctx.save_for_backward(stream, weight)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y, stream

    @staticmethod
    def backward(ctx, dy, dstream):
        if dy is None:  # the addition alone
            return None if dstream is None else dstream.to(BF16), dstream, None, None
        stream, weight = ctx.saved_tensors
        with torch.no_grad():
            grads = _backward(stream, weight, ctx.eps, dy, dstream)
        return _once("the residual norm", (*grads, None), stream, weight, dy, dstream)


def _backward(stream, weight, eps, dy, dstream):
    """(dx, dresidual, dweight)."""
    f32 = stream.dtype == F32
    dx = torch.empty(stream.shape, dtype=BF16, device=stream.device)
    dresidual = torch.empty(stream.shape, dtype=F32, device=stream.device) if f32 else None
    dweight = torch.empty(weight.shape, dtype=F32, device=stream.device)
    if stream.numel() == 0:
        return dx, dresidual if f32 else dx, dweight.zero_()
    s, g, w = _rows(stream), _rows(dy), weight.contiguous()
    h = None if dstream is None else _rows(dstream)
    rows, d = s.shape
    need = _hip.query_on(s, "ws_add_rmsnorm_backward_partial_floats", rows, d)
    partial = torch.empty((need,), dtype=F32, device=s.device) if need else None
    _hip.call_on(s, "ws_add_rmsnorm_backward", s.data_ptr(), int(f32), w.data_ptr(),
                 eps, g.data_ptr(), _row_stride(g), _hip.ptr(h),
                 0 if h is None else _row_stride(h), rows, d, dx.data_ptr(), _hip.ptr(dresidual),
                 dweight.data_ptr(), _hip.ptr(partial))
    return dx, dresidual if f32 else dx, dweight


def _weight(weight: Tensor) -> Tensor:
    """The weight in FP32 (a BF16 one with autograd through the cast)."""
    return weight.float() if weight.dtype == BF16 else weight


def add_rmsnorm(x: Tensor, residual: Tensor, weight: Tensor, eps: float = 1e-5
                ) -> tuple[Tensor, Tensor]:
    """(y, stream) for x [..., d] BF16 and a residual of its shape, BF16 or FP32: stream =
    r(x + residual) in the residual's type, and its RMSNorm y in BF16, with autograd to x, the
    residual and the weight [d] (FP32 or BF16).

    One read of both inputs, one write of both outputs. Statistics, the weight's gradient and all
    products are FP32; y and the gradients are rounded once. Sums of squares have to be in FP32's
    range. Rows of up to 8192 columns, any strides."""
    if not x.is_cuda:
        raise ValueError("Residual norms require CUDA tensors")
    weight = _weight(weight)
    native = _hip.host_ops()
    if native is not None:
        return native.native_add_rmsnorm(x, residual, weight, eps)
    return _add_rmsnorm(x, residual, weight, float(eps))


# (The forms without the C++ operators run eagerly inside a compiled function.)
@torch.compiler.disable
def _add_rmsnorm(x: Tensor, residual: Tensor, weight: Tensor, eps: float) -> tuple[Tensor, Tensor]:
    _check(x, residual, weight)
    _refuse_tangents("add_rmsnorm", x, residual, weight)
    return _AddRmsnorm.apply(x, residual, weight, eps)


def rmsnorm_quantize(x: Tensor, weight: Tensor, eps: float = 1e-5, residual: Tensor | None = None,
                     scale_dtype: torch.dtype = E8M0) -> tuple[Tensor, Tensor, Tensor]:
    """(q, scale, stream) of ``add_rmsnorm``'s y before its rounding: ``quantize_rows`` of it, as
    rows of the last dimension (q [rows, d] e4m3, scale [rows, ceil(d / 128)], for ``fp8_mm``).
    Without a residual the stream is x. A row with an infinity or a NaN has blocks that
    dequantize to NaN. No gradient is recorded, through the stream either."""
    if not x.is_cuda:
        raise ValueError("Residual norms require CUDA tensors")
    if scale_dtype not in _SCALE_TYPES:
        raise ValueError("Scales are torch.float8_e8m0fnu or torch.float32")
    weight, e8m0 = _weight(weight), scale_dtype == E8M0
    native = _hip.host_ops()
    if native is not None:
        q, scale, stream = native.native_rmsnorm_quantize(x, residual, weight, eps, e8m0)
        return q, scale, x.detach() if residual is None else stream
    return _rmsnorm_quantize(x, residual, weight, float(eps), e8m0)


@torch.compiler.disable
def _rmsnorm_quantize(x, residual, weight, eps, e8m0):
    _check(x, residual, weight)
    _refuse_tangents("rmsnorm_quantize", x, residual, weight)
    if x.numel() == 0:
        raise ValueError("Quantization takes non-empty rows")
    x = x.detach()
    a, w = _rows(x), weight.detach().contiguous()
    rows, d = a.shape
    r = stream = None
    if residual is not None:
        r = _rows(residual.detach())
        stream = torch.empty(x.shape, dtype=r.dtype, device=x.device)
    q, scale = _data(rows, d, x.device), _scales(rows, _blocks(d), e8m0, x.device)
    _hip.call_on(x, "ws_rmsnorm_quantize", a.data_ptr(), _row_stride(a), _hip.ptr(r),
                 0 if r is None else _row_stride(r), int(r is not None and r.dtype == F32),
                 w.data_ptr(), eps, rows, d, int(not e8m0), q.data_ptr(), q.shape[1],
                 scale.data_ptr(), scale.shape[1], _hip.ptr(stream))
    return (*_views(q, scale, d, e8m0, rows), x if stream is None else stream)
