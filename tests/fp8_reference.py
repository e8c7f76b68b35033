"""Plain 64-bit restatement of the block quantization and the block-scaled product, written
from their definitions; used by the 8-bit tests."""
import math

import numpy as np
import torch

BLOCK = 128
E8M0, F32 = torch.float8_e8m0fnu, torch.float32


def e4m3_round(x: np.ndarray) -> np.ndarray:
    """The nearest e4m3 value, ties to the even one (|x| <= 464 rounds to at most 448)."""
    mag = np.abs(x)
    with np.errstate(divide="ignore"):
        exponent = np.floor(np.log2(np.where(mag > 0, mag, 1.0)))
    step = 2.0 ** (np.maximum(exponent, -6) - 3)
    return np.round(x / step) * step  # numpy rounds halves to even


def block_scale(amax: float, scale_dtype) -> float:
    if scale_dtype == E8M0:
        if amax == 0.0:
            return 2.0 ** -126
        m, e = math.frexp(amax / 448.0)
        return 2.0 ** max(-126, e - 1 if m == 0.5 else e)
    return float(np.float32(max(amax, 2.0 ** -100)) * (np.float32(1.0) / np.float32(448.0)))


def quantize(x: np.ndarray, scale_dtype, rows_per_block: int = 1):
    """(q, scale) of finite x [M, K] (values of FP32 at most): q as its values in 64 bits."""
    m, k = x.shape
    mb, kb = -(-m // rows_per_block), -(-k // BLOCK)
    q, scale = np.zeros((m, k)), np.zeros((mb, kb))
    for i in range(mb):
        for b in range(kb):
            at = np.s_[i * rows_per_block:(i + 1) * rows_per_block, b * BLOCK:(b + 1) * BLOCK]
            amax = float(np.abs(x[at]).max())
            scale[i, b] = block_scale(amax, scale_dtype)
            if scale_dtype == E8M0:
                scaled = x[at] / scale[i, b]
            else:  # every operation rounded to FP32
                factor = np.float32(1.0) / np.float32(max(amax, 2.0 ** -100)) * np.float32(448.0)
                scaled = (x[at].astype(np.float32) * factor).astype(np.float64)
            q[at] = e4m3_round(scaled)
    return q, scale


def dequantize(q: np.ndarray, scale: np.ndarray) -> np.ndarray:
    rows = 1 if scale.shape[0] == q.shape[0] else BLOCK
    wide = np.repeat(np.repeat(scale, rows, 0), BLOCK, 1)[:q.shape[0], :q.shape[1]]
    return q * wide


def values(t: torch.Tensor) -> np.ndarray:
    """A tensor's values in 64 bits (e4m3, e8m0 bytes as their powers of two, others)."""
    t = t.detach().cpu()
    if t.dtype == E8M0:
        code = t.contiguous().view(torch.uint8).numpy().astype(np.float64)
        return np.where(code == 255, np.nan, 2.0 ** (code - 127))
    return t.float().numpy().astype(np.float64) if t.dtype != torch.float64 else t.numpy()
