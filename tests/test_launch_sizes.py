"""Sizes beyond one launch's 2^32 threads are refused before it (CPU)."""
import pytest

from ops import _hip

P = 1 << 20  # never dereferenced: every call below fails validation first


@pytest.mark.parametrize("rows,cols,form", [(2 ** 31 - 256, 129, 2), (2 ** 30, 256, 1)])
def test_quantization(rows, cols, form):
    with pytest.raises(RuntimeError, match="too many 128 x 128 tiles"):
        _hip.call("ws_fp8_quantize", P, cols, 0, rows, cols, form, 0, P, 256, P, 4, P, 2 ** 31, P, 2 ** 24, None)


def test_pack():
    with pytest.raises(RuntimeError, match="too large"):
        _hip.call("ws_fp8_pack", P, 4096, 1, P, 4096, 2 ** 24, 4096, None)


def test_head_scores():
    with pytest.raises(RuntimeError, match="too many rows"):
        _hip.call("ws_linear_token_scores", P, 64, P, 64, P, 2 ** 26, 50, 64, 1.0, P, P, P, P, None)
