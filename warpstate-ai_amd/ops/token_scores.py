"""Scores of given tokens on gfx950: log probability, entropy and the likeliest tokens.

What scoring, preference and policy training and decoding take from the LM head beside its
cross-entropy (``fused_execution.linear_cross_entropy``; the reference's preference training
forms per-token log probabilities from a chunked head of its own, dpo.py:150-154), with l the
logits over the temperature:

    logprob = l[token] - lse,   lse = log sum_j e^l_j
    entropy = lse - sum_j p_j l_j,   p_j = e^(l_j - lse)

* ``token_scores``: from logits, with the ``top_k`` likeliest tokens and autograd to the
  logits.
* ``linear_token_scores``: from the hidden state and the head weight, with autograd to both; the
  logits exist in registers only, in FP32 (the cross-entropy rounds them to BF16, as the reference's
  training does), and no [rows, vocab] tensor is written but one chunk of BF16 logit gradients.

A token of -100 is ignored: its log probability is 0 and passes no gradient. Its row still has
an entropy, whose gradient it passes. Any other token outside the vocabulary gets NaN (and a
gradient of NaN, unless its log probability's upstream gradient is zero). Logits of -inf have
probability 0.

First derivatives by reverse mode only: forward-mode tensors and functorch's derivatives are
refused, and so is a second differentiation.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from ops import _hip
from ops.fused_execution import TRANSPOSE_MIN_ROWS, transpose

BF16, F32 = torch.bfloat16, torch.float32
Tensor = torch.Tensor
# Logit gradients of one chunk of the backward, BF16: 1 GiB, 16384 rows at a vocabulary of
# 32768. A batch of one chunk writes a BF16 weight's gradient at once, without an FP32 sum beside
# it (scores and gradients of 16384 rows, us, chunks of 8192 / 16384: 2048 over 32768 6426 /
# 6240, 512 over 4096 610 / 399).
CHUNK_LOGITS = 1 << 29
MAX_CHUNK = 2 ** 31 - 1
MAX_TOP_K = 64
MAX_VOCAB = 524288
# 1 / temperature: a normal FP32 number, and finite times log2 e.
INVERSE_RANGE = 2.0 ** -126, 2.3e38


class TokenScores(NamedTuple):
    """Scores of [rows] tokens; the last two are [rows, top_k], largest first."""
    logprob: Tensor
    entropy: Tensor
    top_logprobs: Tensor
    top_ids: Tensor


def _check_tokens(tokens: Tensor, rows: int, device) -> Tensor:
    if tokens.dtype != torch.int64 or tokens.shape != (rows,) or tokens.device != device:
        raise ValueError("Tokens must be an int64 vector, one per row, on the operands' device")
    return tokens.contiguous()


def _inverse(temperature: float) -> float:
    temperature = float(temperature)
    inverse = 1.0 / temperature if temperature else math.inf
    if not INVERSE_RANGE[0] <= inverse <= INVERSE_RANGE[1]:
        raise ValueError(f"The temperature must lie between 4.4e-39 and 8.5e37, not {temperature}")
    return inverse


def _grads(*grads: Tensor | None) -> list[Tensor | None]:
    """Upstream gradients as the kernels read them: contiguous FP32."""
    return [None if g is None else g.to(F32).contiguous() for g in grads]


class _TokenScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k, inv_t):
        rows, vocab = logits.shape
        f32 = dict(dtype=F32, device=logits.device)
        logprob, entropy, lse = torch.empty((3, rows), **f32).unbind()
        top = torch.empty((rows, top_k), **f32)
        ids = torch.empty((rows, top_k), dtype=torch.int64, device=logits.device)
        if rows:
            need = _hip.query_on(logits, "ws_token_scores_workspace_bytes", rows, vocab, top_k)
            work = torch.empty((need,), dtype=torch.uint8, device=logits.device) if need else None
            _hip.call_on(logits, "ws_token_scores", logits.data_ptr(), _row_stride(logits),
                         int(logits.dtype == F32), tokens.data_ptr(), rows, vocab, inv_t, top_k,
                         _hip.ptr(work), lse.data_ptr(), logprob.data_ptr(), entropy.data_ptr(),
                         top.data_ptr(), ids.data_ptr())
        ctx.save_for_backward(logits, tokens, lse, entropy)
        ctx.inv_t = inv_t
        ctx.mark_non_differentiable(top, ids)
        ctx.set_materialize_grads(False)
        return logprob, entropy, top, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogprob, dentropy, _dtop, _dids):
        if dlogprob is None and dentropy is None:
            return None, None, None, None
        logits, tokens, lse, entropy = ctx.saved_tensors
        rows, vocab = logits.shape
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
        if rows:
            g, h = _grads(dlogprob, dentropy)
            _hip.call_on(logits, "ws_token_scores_backward", logits.data_ptr(), _row_stride(logits),
                         int(logits.dtype == F32), tokens.data_ptr(), rows, vocab, ctx.inv_t,
                         lse.data_ptr(), entropy.data_ptr(), _hip.ptr(g), _hip.ptr(h),
                         out.data_ptr(), vocab)
        return out, None, None, None


def _row_stride(t: Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _unit_rows(t: Tensor) -> Tensor:
    """t itself, or a copy, with a unit column stride and rows that do not overlap."""
    rows, cols = t.shape
    if (t.stride(1) == 1 or cols == 1) and (rows <= 1 or t.stride(0) >= cols):
        return t
    return t.contiguous()


def token_scores(logits: Tensor, tokens: Tensor, top_k: int = 0,
                 temperature: float = 1.0) -> TokenScores:
    """Scores of ``tokens`` [rows] under ``logits`` [rows, vocab] (BF16 or FP32, any strides): FP32
    log probabilities and entropies, both differentiable, and the log probabilities and ids of
    the ``top_k`` largest logits (at most 64), equal logits in the order of their ids (not
    differentiable).

    One read of the logits forward, one read and one write backward. A row of -inf only has no
    distribution: its scores are NaN, and its gradient, unless both its upstream gradients are
    zero, whose rows get zeros. NaN or +inf logits make their row's scores NaN and the order of
    its likeliest tokens unspecified. Finite logits have finite scores whatever their size, as
    far as FP32 holds a distance over the temperature: a row masked with its type's lowest value
    throughout is uniform. Vocabularies up to 524288. Under torch.compile it runs
    eagerly (a graph break)."""
    # (Not a decorator of this function, which would add its own calls to each eager one.)
    scores = _eager_token_scores if torch.compiler.is_compiling() else _scores
    return scores(logits, tokens, top_k, temperature)


def _scores(logits: Tensor, tokens: Tensor, top_k: int, temperature: float) -> TokenScores:
    if not logits.is_cuda:
        raise ValueError("Token scores require CUDA tensors")
    native = _hip.host_ops()
    if native is not None:
        return TokenScores(*native.native_token_scores(logits, tokens, top_k, temperature))
    if logits.dtype not in (BF16, F32) or logits.ndim != 2:
        raise ValueError("Expected BF16 or FP32 logits [rows, vocab]")
    rows, vocab = logits.shape
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"Token scores take 1 to {MAX_VOCAB} logits a row, not {vocab}")
    if not 0 <= top_k <= min(MAX_TOP_K, vocab):
        raise ValueError(f"top_k must lie in [0, {min(MAX_TOP_K, vocab)}], not {top_k}")
    tokens = _check_tokens(tokens, rows, logits.device)
    return TokenScores(*_TokenScores.apply(_unit_rows(logits), tokens, int(top_k),
                                           _inverse(temperature)))


_eager_token_scores = torch.compiler.disable(_scores)


def _head_operand(t: Tensor) -> Tensor:
    """A BF16 head operand with 16-byte rows of a multiple of 8: t itself or a copy, padded with
    zeros (which add nothing to a product)."""
    t = t.to(BF16)
    d = t.shape[1]
    if (t.stride(1) == 1 and d % 8 == 0 and t.data_ptr() % 16 == 0
            and (t.shape[0] <= 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= d))):
        return t
    out = torch.zeros((t.shape[0], -(-d // 8) * 8), dtype=BF16, device=t.device)
    out[:, :d].copy_(t)
    return out


class _LinearTokenScores(torch.autograd.Function):
    """Scores from ``_head_operand``'s h and w, with gradients to the tensors they came from."""

    @staticmethod
    def forward(ctx, hidden, weight, h, w, tokens, inv_t, chunk_rows):
        rows, d = h.shape
        vocab = w.shape[0]
        logprob, entropy, lse = torch.empty((3, rows), dtype=F32, device=h.device).unbind()
        if rows:
            need = _hip.query_on(h, "ws_linear_token_scores_workspace_floats", rows, vocab, d)
            work = torch.empty((need,), dtype=F32, device=h.device)
            _hip.call_on(h, "ws_linear_token_scores", h.data_ptr(), _row_stride(h), w.data_ptr(),
                         _row_stride(w), tokens.data_ptr(), rows, vocab, d, inv_t, work.data_ptr(),
                         lse.data_ptr(), logprob.data_ptr(), entropy.data_ptr())
        ctx.save_for_backward(h, w, tokens, lse, entropy)
        ctx.args = (inv_t, chunk_rows, hidden.shape[1], hidden.dtype, weight.dtype)
        ctx.set_materialize_grads(False)
        return logprob, entropy

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogprob, dentropy):
        none = (None,) * 7
        want_h, want_w = ctx.needs_input_grad[:2]
        if (dlogprob is None and dentropy is None) or not (want_h or want_w):
            return none
        h, w, tokens, lse, entropy = ctx.saved_tensors
        inv_t, chunk_rows, width, hidden_dtype, weight_dtype = ctx.args
        rows, d = h.shape
        vocab = w.shape[0]
        dh = torch.empty((rows, d), dtype=BF16, device=h.device) if want_h else None
        # A BF16 weight's gradient is rounded as it is written where one chunk makes all of it.
        bf16 = weight_dtype == BF16 and rows <= chunk_rows and vocab % 8 == 0
        dw = (torch.empty((vocab, d), dtype=BF16 if bf16 else F32, device=h.device) if want_w
              else None)
        if rows:
            g, e = _grads(dlogprob, dentropy)
            need = _hip.query("ws_linear_token_scores_backward_workspace_bytes", rows, vocab, d,
                              chunk_rows)
            work = torch.empty((need,), dtype=torch.uint8, device=h.device)
            # The dHidden product reads the head weight along the vocabulary.
            wt = (transpose(w) if want_h and rows >= TRANSPOSE_MIN_ROWS and vocab % 8 == 0
                  else None)
            _hip.call_on(h, "ws_linear_token_scores_backward", h.data_ptr(), _row_stride(h),
                         w.data_ptr(), _row_stride(w), _hip.ptr(wt), tokens.data_ptr(),
                         lse.data_ptr(), entropy.data_ptr(), _hip.ptr(g), _hip.ptr(e), rows, vocab,
                         d, inv_t, work.data_ptr(), chunk_rows, _hip.ptr(dh), d, _hip.ptr(dw), d,
                         int(bf16))
        elif want_w:
            dw.zero_()
        return (None if dh is None else dh[:, :width].to(hidden_dtype),
                None if dw is None else dw[:, :width].to(weight_dtype), *none[2:])


@torch.compiler.disable
def linear_token_scores(hidden: Tensor, weight: Tensor, tokens: Tensor, temperature: float = 1.0,
                        chunk_rows: int | None = None) -> tuple[Tensor, Tensor]:
    """(logprob, entropy) [rows] FP32 of ``tokens`` under the logits hidden @ weight.T, for hidden
    [rows, d] and the head weight [vocab, d], BF16 or FP32 (rounded to BF16 first, as F.linear
    under BF16 autocast does), with autograd to both.

    The logits are FP32 and never leave the registers. The backward recomputes them
    ``chunk_rows`` rows at a time (None: as many as 1 GiB of BF16 gradients holds); their
    gradient is rounded to BF16 once for the two products, whose sums are FP32, and so is the
    weight's gradient over all chunks. Both gradients come in their operand's type, the hidden
    state's with BF16 precision in either (it is the gradient of the rounded operand). Its
    probabilities are off by up to 2^-24 of the row's log-sum-exp, as the FP32 logits are. Under
    torch.compile it runs eagerly (a graph break)."""
    if not (hidden.is_cuda and weight.is_cuda):
        raise ValueError("Token scores require CUDA tensors")
    if (hidden.ndim != 2 or weight.ndim != 2 or hidden.shape[1] != weight.shape[1]
            or weight.numel() == 0 or hidden.device != weight.device):
        raise ValueError("Expected hidden [rows, d] and weight [vocab, d] on one device")
    if hidden.dtype not in (BF16, F32) or weight.dtype not in (BF16, F32):
        raise ValueError("Head operands are BF16 or FP32")
    if chunk_rows is None:
        chunk_rows = max(256, CHUNK_LOGITS // weight.shape[0] // 256 * 256)
    if chunk_rows < 1:
        raise ValueError("chunk_rows must be positive")
    # (What the backward would refuse: a chunk's rows of logit gradients, padded to whole pieces.)
    chunk, vocab = min(chunk_rows, hidden.shape[0]), weight.shape[0]
    row = -(-vocab // 64) * 64 if vocab % 8 else vocab
    if (chunk * row >= MAX_CHUNK and torch.is_grad_enabled()
            and (hidden.requires_grad or weight.requires_grad)):
        raise ValueError(f"chunk_rows times the vocabulary must be less than {MAX_CHUNK}, not "
                         f"{chunk} x {row}")
    tokens = _check_tokens(tokens, hidden.shape[0], hidden.device)
    native = _hip.host_ops()
    scores = _LinearTokenScores.apply if native is None else native.native_head_scores
    return scores(hidden, weight, _head_operand(hidden.detach()), _head_operand(weight.detach()),
                  tokens, _inverse(temperature), int(chunk_rows))
