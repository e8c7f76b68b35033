"""8-bit projections on gfx950: quantization in blocks of 128 and the block-scaled product.

The 8-bit counterparts of the BF16 projections (``fused_execution.mm``, ``dgrad_mm``,
``mm_f32``; the BF16 step is ops/matmul_execution.py:236-244): operands are e4m3 with one
scale for each block of 128 along the reduction, so that one large feature costs its own
block's small values their precision and no others', and the product accumulates in FP32
across blocks.

* ``quantize_rows``, ``quantize_columns``, ``quantize_rows_and_columns``: an activation or a
  gradient, one scale per 1 x 128 block, as the operand of a product that reduces over its
  columns, its rows (transposed), or both from one read.
* ``quantize_weight``: one scale per 128 x 128 block, so that the same values serve the
  forward product and, transposed, the input gradient.
* ``fp8_mm``: the product of two such matrices.
* ``fp8_linear``: a bias-free projection with autograd, all three products in 8 bits.

Scales are e8m0 (``torch.float8_e8m0fnu``: powers of two, applied by the matrix
instructions themselves, the faster choice) or FP32 (as published 8-bit checkpoints hold them,
applied in FP32 to each block's product). A power of two costs next to nothing: e4m3 is a
floating-point type, so the scale only moves its range, and less than one of its eighteen
binades goes unused.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from ops import _hip
from ops.fused_execution import mm_f32_group

BF16, F32 = torch.bfloat16, torch.float32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BLOCK = 128
Tensor = torch.Tensor

_SCALE_TYPES = (E8M0, F32)
_ROWS, _COLUMNS, _BLOCKS = 1, 2, 4


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _check_input(x: Tensor, scale_dtype: torch.dtype) -> tuple[Tensor, bool]:
    """(x with a unit column stride, whether its scales are e8m0)."""
    if not x.is_cuda:
        raise ValueError("8-bit kernels require CUDA tensors")
    if x.dtype not in (BF16, F32):
        raise ValueError("Quantization takes BF16 or FP32 matrices")
    if x.ndim != 2 or x.numel() == 0:
        raise ValueError("Quantization takes a non-empty matrix")
    if scale_dtype not in _SCALE_TYPES:
        raise ValueError("Scales are torch.float8_e8m0fnu or torch.float32")
    x = x.detach()
    rows, cols = x.shape
    if not (x.stride(1) == 1 or cols == 1) or (rows > 1 and x.stride(0) < cols):
        x = x.contiguous()
    return x, scale_dtype == E8M0


def _ceil(n: int, unit: int) -> int:
    return -(-n // unit) * unit


def _data(rows: int, cols: int, device) -> Tensor:
    """Uninitialised bytes for e4m3 [rows, cols] over rows of a multiple of 16 bytes."""
    return torch.empty((rows, _ceil(cols, 16)), dtype=torch.uint8, device=device)


def _scales(rows: int, blocks: int, e8m0: bool, device) -> Tensor:
    """Uninitialised scales [rows, blocks] in the layout the product reads: e8m0 bytes, rows
    of a multiple of four; FP32, one column of all rows' scales (a multiple of four) per block."""
    if e8m0:
        return torch.empty((rows, _ceil(blocks, 4)), dtype=torch.uint8, device=device)
    return torch.empty((blocks, _ceil(rows, 4)), dtype=F32, device=device)


def _quantize(x: Tensor, e8m0: bool, form: int, transposed: bool = False):
    """(q, scale, qt, scale_t) as the kernel's whole buffers (``_data``, ``_scales``), None for
    the forms that are not wanted."""
    native = _hip.host_ops()
    if native is not None:
        q, scale, qt, scale_t = native.native_quantize(x, e8m0, form, transposed)
        return (*((q, scale) if form != _COLUMNS else (None, None)),
                *((qt, scale_t) if form & _COLUMNS or transposed else (None, None)))
    rows, cols = x.shape
    row_blocks, col_blocks = _blocks(rows), _blocks(cols)
    q = scale = qt = scale_t = None
    if form != _COLUMNS:
        q = _data(rows, cols, x.device)
        scale = _scales(row_blocks if form == _BLOCKS else rows, col_blocks, e8m0, x.device)
    if form & _COLUMNS or transposed:
        qt = _data(cols, rows, x.device)
        scale_t = _scales(col_blocks if form == _BLOCKS else cols, row_blocks, e8m0, x.device)
    _hip.call_on(x, "ws_fp8_quantize", x.data_ptr(), x.stride(0) if rows > 1 else cols,
                 int(x.dtype == F32), rows, cols, form, int(not e8m0), _hip.ptr(q),
                 0 if q is None else q.shape[1], _hip.ptr(scale),
                 0 if scale is None else scale.shape[1], _hip.ptr(qt),
                 0 if qt is None else qt.shape[1], _hip.ptr(scale_t),
                 0 if scale_t is None else scale_t.shape[1])
    return q, scale, qt, scale_t


def _views(q: Tensor, scale: Tensor, cols: int, e8m0: bool, scale_rows: int
           ) -> tuple[Tensor, Tensor]:
    """The e4m3 matrix and its scales [scale_rows, blocks] in a pair of whole buffers."""
    blocks = _blocks(cols)
    q = q.view(E4M3)
    if q.shape[1] != cols:
        q = q[:, :cols]
    if e8m0:
        scale = scale.view(E8M0)
        return q, scale if scale.shape[1] == blocks else scale[:, :blocks]
    return q, scale[:, :scale_rows].T


def quantize_rows(x: Tensor, scale_dtype: torch.dtype = E8M0) -> tuple[Tensor, Tensor]:
    """(q, scale) of x [M, K] (BF16 or FP32): q [M, K] e4m3, scale [M, ceil(K / 128)], so that
    q times its block's scale is x to e4m3's precision. The scale of a block with largest
    magnitude amax is the least power of two 2^e >= amax / 448 (e >= -126), or
    max(amax, 2^-100) / 448 in FP32. A block that holds an infinity or a NaN dequantizes to
    NaN, all of it. Another block's zeros stay zeros."""
    native = _hip.host_ops()
    if native is not None and x.is_cuda and scale_dtype in _SCALE_TYPES:
        return native.native_quantize_rows(x.detach() if x.requires_grad else x,
                                           scale_dtype == E8M0)
    x, e8m0 = _check_input(x, scale_dtype)
    q, scale = _quantize(x, e8m0, _ROWS)[:2]
    return _views(q, scale, x.shape[1], e8m0, x.shape[0])


def quantize_columns(x: Tensor, scale_dtype: torch.dtype = E8M0) -> tuple[Tensor, Tensor]:
    """(qt, scale_t) of x [M, K]: ``quantize_rows`` of x.T, qt [K, M] written transposed and
    scale_t [K, ceil(M / 128)]: the operand of a product that reduces over the rows of x."""
    x, e8m0 = _check_input(x, scale_dtype)
    qt, scale_t = _quantize(x, e8m0, _COLUMNS)[2:]
    return _views(qt, scale_t, x.shape[0], e8m0, x.shape[1])


def quantize_rows_and_columns(x: Tensor, scale_dtype: torch.dtype = E8M0
                              ) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(q, scale, qt, scale_t): ``quantize_rows`` and ``quantize_columns`` from one read of x."""
    x, e8m0 = _check_input(x, scale_dtype)
    rows, cols = x.shape
    q, scale, qt, scale_t = _quantize(x, e8m0, _ROWS | _COLUMNS)
    return (*_views(q, scale, cols, e8m0, rows), *_views(qt, scale_t, rows, e8m0, cols))


def quantize_weight(weight: Tensor, scale_dtype: torch.dtype = E8M0
                    ) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(q, scale, qt, scale_t) of a weight [N, K] (nn.Linear layout, BF16 or FP32) with one
    scale per 128 x 128 block: q [N, K], scale [ceil(N / 128), ceil(K / 128)], and the same
    values transposed, qt [K, N] with scale_t [ceil(K / 128), ceil(N / 128)], for the input
    gradient."""
    weight, e8m0 = _check_input(weight, scale_dtype)
    n, k = weight.shape
    q, scale, qt, scale_t = _quantize(weight, e8m0, _BLOCKS, True)
    return (*_views(q, scale, k, e8m0, _blocks(n)), *_views(qt, scale_t, n, e8m0, _blocks(k)))


def _operand(q: Tensor) -> Tensor:
    """q with rows of whole 16-byte pieces as the product's loads read them: q itself, or a
    zero-padded copy (a reduction that is no multiple of 16, other strides, an unaligned
    view)."""
    rows, k = q.shape
    if (q.stride(1) == 1 and k % 16 == 0 and q.data_ptr() % 16 == 0
            and (rows == 1 or (q.stride(0) % 16 == 0 and q.stride(0) >= k))):
        return q
    if min(q.stride()) < 1:  # an expanded matrix
        q = q.view(torch.uint8).contiguous()
    out = _data(rows, k, q.device)
    _hip.call_on(q, "ws_fp8_pack", q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(),
                 out.shape[1], rows, k)
    return out


def _scale(scale: Tensor, q: Tensor, dtype: torch.dtype, vector: bool, name: str
           ) -> tuple[Tensor, int, int]:
    """(scale, leading dimension, operand rows per scale row) in the layout the product reads;
    scales that lie otherwise are copied. ``vector``: read four rows' FP32 scales at a time."""
    rows, blocks = q.shape[0], _blocks(q.shape[1])
    if scale.dtype != dtype or scale.device != q.device or scale.ndim != 2:
        raise ValueError(f"{name} must be a matrix of {str(dtype).removeprefix('torch.')} scales "
                         f"on {q.device}")
    n, block_rows = scale.shape[0], 1
    if scale.shape != (rows, blocks):
        block_rows = BLOCK
        if scale.shape != (_blocks(rows), blocks):
            raise ValueError(f"{name} must have one scale per row or per 128 rows and one per "
                             f"128 columns, {[rows, blocks]} or {[_blocks(rows), blocks]}, not "
                             f"{list(scale.shape)}")
    s0, s1 = scale.stride()
    size, first = scale.untyped_storage().nbytes(), scale.storage_offset()
    if dtype == E8M0:
        # The kernel reads whole dwords of a row.
        ld = s0 if n > 1 else _ceil(blocks, 4)
        if ((s1 == 1 or blocks == 1) and ld % 4 == 0 and ld >= blocks
                and scale.data_ptr() % 4 == 0
                and first + (n - 1) * ld + _ceil(blocks, 4) <= size):
            return scale, ld, block_rows
        copy = _scales(n, blocks, True, scale.device)
        copy[:, :blocks].copy_(scale.view(torch.uint8))
    else:
        ld = s1 if blocks > 1 else _ceil(n, 4)
        if ((s0 == 1 or n == 1) and ld >= n
                and (not vector or (ld % 4 == 0 and scale.data_ptr() % 16 == 0
                                    and 4 * (first + (blocks - 1) * ld + _ceil(n, 4)) <= size))):
            return scale, ld, block_rows
        copy = _scales(n, blocks, False, scale.device)
        copy[:, :n].copy_(scale.T)
    return copy, copy.shape[1], block_rows


def _check_operand(q: Tensor, name: str) -> None:
    if not q.is_cuda:
        raise ValueError("8-bit kernels require CUDA tensors")
    if q.dtype != E4M3 or q.ndim != 2 or q.numel() == 0:
        raise ValueError(f"{name} must be a non-empty float8_e4m3fn matrix")


def _launch(a: Tensor, lda: int, sa: Tensor, ld_sa: int, rows_a: int, b: Tensor, ldb: int,
            sb: Tensor, ld_sb: int, rows_b: int, e8m0: bool, out: Tensor, k: int) -> None:
    (m, n), k16 = out.shape, _ceil(k, 16)
    need = _hip.query_on(a, "ws_fp8_mm_workspace_bytes", m, n, k16, rows_b, int(not e8m0))
    work = torch.empty((need,), dtype=torch.uint8, device=a.device) if need else None
    _hip.call_on(a, "ws_fp8_mm", a.data_ptr(), lda, sa.data_ptr(), ld_sa, rows_a, b.data_ptr(), ldb,
                 sb.data_ptr(), ld_sb, rows_b, int(not e8m0), out.data_ptr(),
                 out.stride(0) if m > 1 else n, m, n, k16, _hip.ptr(work))


def fp8_mm(a: Tensor, a_scale: Tensor, b: Tensor, b_scale: Tensor,
           out: Tensor | None = None) -> Tensor:
    """C [M, N] = dequantized(a) @ dequantized(b).T in BF16 for e4m3 a [M, K] and b [N, K]
    (nn.Linear layout).

    A scale matrix has one column per 128 columns of its operand and one row per operand row
    or per 128 of them; both are e8m0 or both FP32. Sums are FP32, except that the matrix
    instruction adds groups of eight products after cutting each to 13 bits below the
    group's largest: an error of at most 2^-10 of the sum of the products' magnitudes,
    about 1e-4 of the result's size for random operands, a twentieth of its BF16 rounding. That is why
    there is no FP32 result. ``out`` (BF16, unit column stride) receives the result instead of
    a new tensor. Operands in other layouts than rows of whole 16-byte pieces, and scales in
    other layouts than ``quantize_rows`` gives, are copied first: on every call, for a reduction
    that is no multiple of 16 (one row through 2048 x 5632 takes 12.6 us, through 2048 x 5624 27; through
    11264 x 2040 42). A program that multiplies by one weight many times pads its reduction with
    zeros before ``quantize_weight``. FP32 scales' products have to be in FP32's range. No gradient
    is recorded."""
    native = _hip.host_ops()
    if native is not None and out is None and a.is_cuda:
        return native.native_fp8_mm(a, a_scale, b, b_scale)
    for q, name in ((a, "a"), (b, "b")):
        _check_operand(q, name)
    (m, k), n = a.shape, b.shape[0]
    if b.shape[1] != k or a.device != b.device:
        raise ValueError(f"Expected a [M, K] and b [N, K] on one device, got {list(a.shape)} and "
                         f"{list(b.shape)}")
    if a_scale.dtype not in _SCALE_TYPES:
        raise ValueError("Scales are torch.float8_e8m0fnu or torch.float32")
    if out is None:
        out = torch.empty((m, n), dtype=BF16, device=a.device)
    elif out.shape != (m, n) or out.device != a.device or out.dtype != BF16:
        raise ValueError(f"out must be a BF16 tensor of shape {[m, n]} on {a.device}")
    elif (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
        raise ValueError("out must have a unit column stride")
    dtype = a_scale.dtype
    sa, ld_sa, rows_a = _scale(a_scale, a, dtype, False, "a_scale")
    by_rows = b_scale.ndim == 2 and b_scale.shape[0] == n
    sb, ld_sb, rows_b = _scale(b_scale, b, dtype, by_rows, "b_scale")
    a, b = _operand(a), _operand(b)
    wide = _ceil(k, 16)
    _launch(a, a.stride(0) if m > 1 else wide, sa, ld_sa, rows_a, b, b.stride(0) if n > 1 else wide,
            sb, ld_sb, rows_b, dtype == E8M0, out, k)
    return out


def _mm_buffers(q, scale, rows_a, b, b_scale, rows_b, e8m0, out, k):
    """``fp8_mm`` on the whole buffers of ``_quantize``."""
    _launch(q, q.shape[1], scale, scale.shape[1], rows_a, b, b.shape[1], b_scale, b_scale.shape[1],
            rows_b, e8m0, out, k)
    return out


# --- a projection with autograd ------------------------------------------------------------

@torch.library.custom_op("warpstate::fp8_linear", mutates_args=())
def _fp8_linear(x: Tensor, weight: Tensor, e8m0: bool, keep_x: bool, keep_w: bool
                ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(y, qt, qt_scale, wt, wt_scale) for rows x [M, K] BF16 and a weight [N, K]: y [M, N]
    BF16, and the 8-bit operands of the backward's products (empty unless kept): x by columns
    for dW, the weight transposed for dX."""
    m, k = x.shape
    n = weight.shape[0]
    w, w_scale, wt, wt_scale = _quantize(weight, e8m0, _BLOCKS, keep_w)
    q, scale, qt, qt_scale = _quantize(x, e8m0, _ROWS | _COLUMNS if keep_x else _ROWS)
    y = torch.empty((m, n), dtype=BF16, device=x.device)
    _mm_buffers(q, scale, 1, w, w_scale, BLOCK, e8m0, y, k)
    kept = [t if t is not None else x.new_empty((0, 0), dtype=torch.uint8)
            for t in (qt, qt_scale, wt, wt_scale)]
    return (y, *kept)


@_fp8_linear.register_fake
def _fp8_linear_fake(x, weight, e8m0, keep_x, keep_w):
    m, k = x.shape
    n = weight.shape[0]

    def buffers(keep, rows, cols, scale_rows):
        if not keep:
            return x.new_empty((0, 0), dtype=torch.uint8), x.new_empty((0, 0), dtype=torch.uint8)
        blocks = _blocks(cols)
        return (x.new_empty((rows, _ceil(cols, 16)), dtype=torch.uint8),
                x.new_empty((scale_rows, _ceil(blocks, 4)), dtype=torch.uint8) if e8m0 else
                x.new_empty((blocks, _ceil(scale_rows, 4)), dtype=F32))

    return (x.new_empty((m, n)), *buffers(keep_x, k, m, k), *buffers(keep_w, k, n, _blocks(k)))


@torch.library.custom_op("warpstate::fp8_linear_backward", mutates_args=())
def _fp8_linear_backward(grad: Tensor, x: Tensor, qt: Tensor, qt_scale: Tensor, wt: Tensor,
                         wt_scale: Tensor, k: int, e8m0: bool, want_x: bool, want_w: bool,
                         master: bool) -> tuple[Tensor, Tensor]:
    """(dx, dw), each empty unless wanted: dx = q(grad) @ q(W) in BF16; dw of a BF16 weight
    q(grad)^T @ q(x) in BF16, of an FP32 master grad^T @ x with FP32 sums."""
    grad = grad.contiguous()
    m, n = grad.shape
    form = (_ROWS if want_x else 0) | (_COLUMNS if want_w and not master else 0)
    if form:
        g, g_scale, gt, gt_scale = _quantize(grad, e8m0, form)
    dx = torch.empty((m, k) if want_x else (0,), dtype=BF16, device=grad.device)
    if want_x:
        _mm_buffers(g, g_scale, 1, wt, wt_scale, BLOCK, e8m0, dx, n)
    if want_w and master:
        # The entry point that the native kernel calls, so that sums are taken in one order.
        return dx, mm_f32_group([(grad.T, x)], round_bf16=False)[0]
    dw = torch.empty((n, k) if want_w else (0,), dtype=F32 if master else BF16, device=grad.device)
    if want_w:
        _mm_buffers(gt, gt_scale, 1, qt, qt_scale, 1, e8m0, dw, m)
    return dx, dw


@_fp8_linear_backward.register_fake
def _fp8_linear_backward_fake(grad, x, qt, qt_scale, wt, wt_scale, k, e8m0, want_x, want_w, master):
    m, n = grad.shape
    return (grad.new_empty((m, k) if want_x else (0,)),
            grad.new_empty((n, k) if want_w else (0,), dtype=F32 if master else BF16))


def _linear_setup(ctx, inputs, output):
    x, weight, e8m0, keep_x, _keep_w = inputs
    # x itself only where its weight gradient reads it.
    master = weight.dtype == F32
    kept_x = x if master and weight.requires_grad else output[1]
    ctx.save_for_backward(kept_x, *output[1:])
    ctx.set_materialize_grads(False)
    ctx.args = (x.shape[1], e8m0, x.requires_grad, weight.requires_grad, master)


def _linear_autograd(ctx, grad, *_buffers):
    k, e8m0, want_x, want_w, master = ctx.args
    if grad is None:
        return None, None, None, None, None
    dx, dw = _fp8_linear_backward(grad, *ctx.saved_tensors, k, e8m0, want_x, want_w, master)
    return dx if want_x else None, dw if want_w else None, None, None, None


_fp8_linear.register_autograd(_linear_autograd, setup_context=_linear_setup)

_hip.host_ops()


def _refuse_tangents(*tensors: Tensor) -> None:
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("fp8_linear has no forward-mode derivative")


def fp8_linear(x: Tensor, weight: Tensor, scale_dtype: torch.dtype = E8M0) -> Tensor:
    """x @ weight.T of a bias-free projection in 8 bits, with autograd: x [..., K] BF16, weight
    [N, K] (nn.Linear layout), BF16 or an FP32 master.

    y = q(x) q(W)^T and dx = q(dy) q(W) are BF16, of e4m3 operands: W in 128 x 128 blocks, x
    and dy in 1 x 128 blocks along the reduction. A BF16 weight's gradient is in 8 bits too,
    r(q(dy)^T q(x)) with both operands quantized by columns; a step then keeps one byte per
    element of x and of W for the backward. An FP32 master's gradient is FP32, and the 8-bit
    matrix instruction's sums are not (``fp8_mm``): it is dy^T x of the BF16 tensors with FP32
    sums (``mm_f32_group``), from x itself, which costs several times as much where N or K is no
    multiple of 8 (4096 rows, forward and gradients: 1280 x 4480 156 us, 1285 x 4477 603).

    First derivatives by reverse mode only (forward-mode tensors and functorch's derivatives are
    refused)."""
    if x.dtype != BF16:
        raise ValueError("An 8-bit projection takes BF16 activations")
    if x.ndim < 1 or weight.ndim != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"Expected x [..., K] and weight [N, K], got {list(x.shape)} and "
                         f"{list(weight.shape)}")
    if x.device != weight.device:
        raise ValueError("x and weight must be on one device")
    rows = x.reshape(-1, x.shape[-1])
    _check_input(rows, scale_dtype)
    _check_input(weight, scale_dtype)
    if not torch.compiler.is_compiling() and _hip.host_ops() is None:
        _refuse_tangents(x, weight)  # as the native autograd kernel does
    grad = torch.is_grad_enabled()
    y = _fp8_linear(rows.contiguous(), weight.contiguous(), scale_dtype == E8M0,
                    grad and weight.requires_grad and weight.dtype == BF16,
                    grad and x.requires_grad)[0]
    return y.view(*x.shape[:-1], weight.shape[0])
