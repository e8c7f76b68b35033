"""Embedding lookup with scaling on gfx950, with the table's gradient by sorted tokens.

The reference looks tokens up in the FP32 master table (warpstate/model.py:282,307) or, on a BF16
residual stream, in a BF16 copy of the whole table made for every call
(ops/residual_experiment.py:25-58). ``embedding`` reads only the tokens' rows of either table
and rounds what it has read:

    y[t] = r(scale W[token t]),   dW[v] = scale sum over t with token t = v of dy[t]

The gradient's sums are FP32, whatever the types, and their order is fixed by the tokens alone, so
that two calls give the same bits. ``embedding_accumulate_`` adds the gradient to an FP32 buffer
that is there already, such as a tied head's (``fused_execution.linear_cross_entropy_backward``),
and touches the tokens' rows only.

A token of -100 is ignored, as the losses and scores do: its row is zeros, and it takes no
gradient. Any other token outside the vocabulary gets a row of NaN, and takes none either. First
derivatives by reverse mode only: forward-mode tensors and functorch's derivatives are refused,
and so is a second differentiation.
"""

from __future__ import annotations

import math
from ctypes import c_float

import torch

from ops import _hip
from ops.residual_norm import _once, _refuse_tangents, _row_stride, _rows

BF16, F32 = torch.bfloat16, torch.float32
Tensor = torch.Tensor
_WRITE_BF16, _WRITE_F32, _ADD_F32 = 0, 1, 2


def _check_scale(scale: float) -> None:
    if not math.isfinite(c_float(scale).value):  # (the kernels multiply in FP32)
        raise ValueError(f"The scale must be finite in FP32, not {scale}")


def _check(tokens: Tensor, table: Tensor, scale: float) -> None:
    if tokens.dtype != torch.int64 or tokens.device != table.device:
        raise ValueError("Tokens must be int64 on the table's device")
    if table.dtype not in (BF16, F32) or table.ndim != 2 or table.numel() == 0:
        raise ValueError("Expected a non-empty BF16 or FP32 table [vocab, d]")
    _check_scale(scale)


def _sums(dy: Tensor, tokens: Tensor, scale: float, out: Tensor, mode: int) -> None:
    """The sums of dy by token into ``out`` [vocab, d]."""
    tokens = tokens.contiguous()
    rows, (vocab, d) = tokens.numel(), out.shape
    g = _rows(dy) if rows else None
    need = _hip.query("ws_embedding_backward_workspace_bytes", rows, vocab, d)
    work = torch.empty((need,), dtype=torch.uint8, device=out.device) if need else None
    _hip.call_on(out, "ws_embedding_backward", _hip.ptr(g), _row_stride(g) if rows else 0,
                 int(dy.dtype == F32), tokens.data_ptr(), rows, vocab, d, scale, out.data_ptr(),
                 _row_stride(out), mode, _hip.ptr(work))


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table_in, scale, f32):
        tokens, table = tokens.contiguous(), _rows(table_in)
        vocab, d = table.shape
        y = torch.empty((*tokens.shape, d), dtype=F32 if f32 else BF16, device=table.device)
        _hip.call_on(table, "ws_embedding", table.data_ptr(), _row_stride(table),
                     int(table.dtype == F32), tokens.data_ptr(), tokens.numel(), vocab, d, scale,
                     y.data_ptr(), int(f32))
        ctx.save_for_backward(tokens)
        ctx.args = (vocab, d, scale, table.dtype)
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None
        vocab, d, scale, dtype = ctx.args
        out = torch.empty((vocab, d), dtype=dtype, device=dy.device)
        _sums(dy.detach(), ctx.saved_tensors[0], scale, out,
              _WRITE_F32 if dtype == F32 else _WRITE_BF16)
        return _once("the embedding", (None, out, None, None), dy)


def embedding(tokens: Tensor, table: Tensor, scale: float = 1.0,
              out_dtype: torch.dtype = BF16) -> Tensor:
    """scale * table[tokens] for int64 tokens of any shape and a table [vocab, d] (BF16 or an FP32
    master, any strides), in ``out_dtype`` (BF16 or FP32), with autograd to the table.

    Each row is scaled in FP32 and rounded once. The gradient comes in the table's type from FP32
    sums, all of it written (rows without tokens are zeros). Up to 2^22 rows of 2^20
    columns and 2^24 tokens."""
    if not table.is_cuda:
        raise ValueError("Embeddings require CUDA tensors")
    if out_dtype not in (BF16, F32):
        raise ValueError("Embeddings come in BF16 or FP32")
    native = _hip.host_ops()
    if native is not None:
        return native.native_embedding(tokens, table, scale, out_dtype == F32)
    return _embedding(tokens, table, float(scale), out_dtype == F32)


# (Without the C++ operators it runs eagerly inside a compiled function.)
@torch.compiler.disable
def _embedding(tokens: Tensor, table: Tensor, scale: float, f32: bool) -> Tensor:
    _check(tokens, table, scale)
    _refuse_tangents("embedding", table)
    return _Embedding.apply(tokens, table, scale, f32)


def _written(t: Tensor) -> None:
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


@torch.compiler.disable
@torch.no_grad()
def embedding_accumulate_(gradient: Tensor, tokens: Tensor, dy: Tensor, scale: float = 1.0
                          ) -> Tensor:
    """gradient += scale * the sums of dy [..., d] (BF16 or FP32) by token, for an FP32 gradient
    [vocab, d] with a unit column stride. Rows without tokens are neither read nor written.
    Returns the gradient; no graph is recorded. Under torch.compile it runs eagerly (a graph
    break)."""
    if not gradient.is_cuda:
        raise ValueError("Embeddings require CUDA tensors")
    native = _hip.host_ops()
    if native is not None:
        native.native_embedding_accumulate_(gradient, tokens, dy, scale)
        _written(gradient)
        return gradient
    if (gradient.dtype != F32 or gradient.ndim != 2 or gradient.numel() == 0
            or (gradient.stride(1) != 1 and gradient.shape[1] != 1)
            or (gradient.shape[0] > 1 and gradient.stride(0) < gradient.shape[1])):
        raise ValueError("The gradient must be a non-empty FP32 matrix with a unit column stride")
    if tokens.dtype != torch.int64 or tokens.device != gradient.device:
        raise ValueError("Tokens must be int64 on the gradient's device")
    shape = (*tokens.shape, gradient.shape[1])
    if dy.dtype not in (BF16, F32) or dy.shape != shape or dy.device != gradient.device:
        raise ValueError(f"Expected BF16 or FP32 rows of shape {list(shape)} on "
                         f"{gradient.device}")
    _check_scale(scale)
    _sums(dy, tokens, float(scale), gradient, _ADD_F32)
    _written(gradient)
    return gradient
