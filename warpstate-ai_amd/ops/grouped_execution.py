"""Products grouped by expert on gfx950: a projection whose rows each have one of several weights.

The grouped form of the BF16 projections (``fused_execution.mm``, ``dgrad_mm``,
``mm_f32_group``; the BF16 step is ops/matmul_execution.py:236-244). Rows are sorted by expert, and
``offsets`` says where each expert's begin:

    y[t] = r(x[t] W_e^T)   for offsets[e] <= t < offsets[e + 1]

with dx[t] = r(dy[t] W_e) and dW_e = sum over those t of dy[t]^T x[t]. The offsets stay on the
device: nothing waits for them on the host, and a call can be captured and replayed with others.
Experts without rows, and one with all of them, are ordinary cases. The same call serves
low-rank factors of many requests: rows sorted by request, one small weight each.

First derivatives by reverse mode only: forward-mode tensors and functorch's derivatives are
refused, and so is a second differentiation.
"""

from __future__ import annotations

import torch

from ops import _hip
from ops.residual_norm import _once, _refuse_tangents, _row_stride

BF16, F32 = torch.bfloat16, torch.float32
Tensor = torch.Tensor
_NT, _NN = 0, 1


def _check(x: Tensor, weight: Tensor, offsets: Tensor) -> None:
    if x.dtype != BF16 or x.ndim != 2:
        raise ValueError("Grouped products take BF16 rows [rows, k]")
    if (weight.dtype not in (BF16, F32) or weight.ndim != 3 or weight.numel() == 0
            or weight.shape[2] != x.shape[1] or weight.device != x.device):
        raise ValueError(f"Expected non-empty BF16 or FP32 weights [groups, n, {x.shape[1]}] on "
                         f"{x.device}")
    if (offsets.dtype != torch.int64 or offsets.shape != (weight.shape[0] + 1,)
            or offsets.device != x.device):
        raise ValueError("Offsets must be an int64 vector, one more than the groups, on "
                         f"{x.device}")


def _whole_rows(t: Tensor) -> bool:
    """Whether t's rows lie on whole 16-byte pieces and do not overlap."""
    if t.shape[-1] % 8 or (t.stride(-1) != 1 and t.shape[-1] != 1) or t.storage_offset() % 8:
        return False
    inner = t.shape[-1]
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size > 1 and (stride % 8 or stride < inner):
            return False
        inner = size * stride
    return True


def _copy_rows(t: Tensor, rows: int, cols: int, dtype: torch.dtype) -> Tensor:
    """t [rows, cols] or [groups, rows, cols] in other sizes, padded with zeros or cut off."""
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        t = t.contiguous()
    groups = t.shape[0] if t.ndim == 3 else 1
    out = torch.empty((*t.shape[:-2], rows, cols), dtype=dtype, device=t.device)
    _hip.call_on(t, "ws_copy_rows", t.data_ptr(), int(t.dtype == F32),
                 t.stride(0) if t.ndim == 3 else 0, t.stride(-2), t.shape[-2], t.shape[-1],
                 out.data_ptr(), int(dtype == F32), rows * cols, cols, rows, cols, groups)
    return out


def _operand(t: Tensor) -> Tensor:
    """A BF16 operand with 16-byte rows of a multiple of 8: t itself, or a copy whose rows are
    padded with zeros."""
    if _whole_rows(t):
        return t.to(BF16)
    return _copy_rows(t, t.shape[-2], _up(t.shape[-1]), BF16)


def _up(n: int) -> int:
    return -(-n // 8) * 8


def _product(x: Tensor, w: Tensor, offsets: Tensor, form: int) -> Tensor:
    """On operands of ``_operand``: columns up to the next multiple of 8."""
    rows, (groups, n, k) = x.shape[0], w.shape
    if form == _NN:
        n, k = k, n
    y = torch.empty((rows, _up(n)), dtype=BF16, device=x.device)
    need = _hip.query_on(x, "ws_grouped_workspace_floats", rows, groups, n, k, form)
    work = torch.empty((need,), dtype=F32, device=x.device) if need else None
    _hip.call_on(x, "ws_grouped_mm", x.data_ptr(), _row_stride(x), w.data_ptr(),
                 w.stride(1) if w.shape[1] > 1 else w.shape[2], w.stride(0) if groups > 1 else 0,
                 form, offsets.data_ptr(), groups, rows, n, k, y.data_ptr(), y.shape[1],
                 _hip.ptr(work))
    return y


def _first(t: Tensor, cols: int) -> Tensor:
    """The first of t's padded columns."""
    return t if t.shape[-1] == cols else _copy_rows(t, t.shape[-2], cols, t.dtype)


class _GroupedMm(torch.autograd.Function):
    """Of ``_operand``'s a and w, with gradients to the tensors x and weight, which they came from. Kept
    is what these read: dx the weights, dW the rows. ``inputs``: tensors without elements that depend
    on x and weight."""

    @staticmethod
    def forward(ctx, x, weight, a, w, offsets, inputs):
        want_x, want_w = ctx.needs_input_grad[:2]
        ctx.save_for_backward(a if want_w else None, w if want_x else None, offsets, *inputs)
        ctx.args = (weight.shape[1], x.shape[1], weight.dtype)
        ctx.set_materialize_grads(False)
        return _first(_product(a, w, offsets, _NT), weight.shape[1])

    @staticmethod
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None, None, None
        a, w, offsets, *inputs = ctx.saved_tensors
        n, k, dtype = ctx.args
        dx = dw = None
        with torch.no_grad():
            g = _operand(dy)
            if ctx.needs_input_grad[0]:
                dx = _first(_product(g, w, offsets, _NN), k)
            if ctx.needs_input_grad[1]:
                groups = offsets.shape[0] - 1
                dw = torch.empty((groups, n, a.shape[1]), dtype=dtype, device=a.device)
                _hip.call_on(a, "ws_grouped_weight_grad", g.data_ptr(), _row_stride(g),
                             a.data_ptr(), _row_stride(a), offsets.data_ptr(), groups, a.shape[0], n,
                             a.shape[1], dw.data_ptr(), int(dtype == F32))
                dw = _first(dw, k)
        return _once("a grouped product", (dx, dw, None, None, None, None), *inputs, dy)


def grouped_mm(x: Tensor, weight: Tensor, offsets: Tensor) -> Tensor:
    """y [rows, n] BF16 for BF16 rows x [rows, k], weights [groups, n, k] (nn.Linear layout for each
    group; BF16, or FP32 masters, rounded to BF16 first as F.linear under BF16 autocast does) and
    int64 ``offsets`` [groups + 1] on the device: rows offsets[e] to offsets[e + 1] are multiplied
    by weight e. With autograd to x (BF16) and the weights (their type, from FP32 sums). Up to 16384
    groups and 2^30 rows; in tiles of 256 x 256, fewer than 2^24 of the result (and of x's gradient: of
    (rows / 256 + groups + 2) ceil(n / 256)) and fewer than 2^22 of the weights. A call whose gradients
    would pass that is refused where it is recorded.

    Offsets must not decrease; rows before the first and behind the last get zeros, in y and in the
    gradient of x. No value of theirs leads an access out of the operands, but rows that
    decreasing ones name twice or not at all are unspecified. Sums are FP32. A row's bits depend on the
    kernel that the sizes choose, not on the other rows' values. Operands whose rows are not whole
    16-byte pieces (weights or rows with k no multiple of 8, other strides) are copied first, on
    every call: a program that uses such weights many times pads their rows once. BF16 weights are
    read as they are where there are few rows and no gradients."""
    if not x.is_cuda:
        raise ValueError("Grouped products require CUDA tensors")
    native = _hip.host_ops()
    if native is not None:
        return native.native_grouped_mm(x, weight, offsets)
    return _grouped_mm(x, weight, offsets)


# (Without the C++ operators it runs eagerly inside a compiled function.)
@torch.compiler.disable
def _grouped_mm(x: Tensor, weight: Tensor, offsets: Tensor) -> Tensor:
    _check(x, weight, offsets)
    _refuse_tangents("grouped_mm", x, weight)
    inputs = ()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        _hip.call("ws_grouped_backward_check", x.shape[0], *weight.shape, int(x.requires_grad),
                  int(weight.requires_grad), int(weight.dtype == F32))
        # (Copies: a view would keep the whole of its tensor.)
        inputs = tuple(t[:0].clone() for t in (x, weight) if t.requires_grad)
    return _GroupedMm.apply(x, weight, _operand(x.detach()), _operand(weight.detach()),
                            offsets.contiguous(), inputs)
