"""What the 8-bit entry points refuse, before any launch (CPU)."""
import pytest
import torch

from ops import _hip
from ops import fp8_execution as fp8

E8M0, F32, E4M3 = torch.float8_e8m0fnu, torch.float32, torch.float8_e4m3fn
P = 1 << 20  # never dereferenced: every call below fails validation first


@pytest.mark.parametrize("call", [fp8.quantize_rows, fp8.quantize_columns, fp8.quantize_weight,
                                  fp8.quantize_rows_and_columns])
def test_quantization_needs_the_gpu(call):
    with pytest.raises(ValueError, match="CUDA"):
        call(torch.zeros(4, 4, dtype=torch.bfloat16))


def test_product_and_projection_need_the_gpu():
    q = torch.zeros(4, 16, dtype=torch.uint8).view(E4M3)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.fp8_mm(q, torch.ones(4, 1), q, torch.ones(4, 1))
    with pytest.raises(ValueError, match="CUDA"):
        fp8.fp8_linear(torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(8, 16))
    with pytest.raises(ValueError, match="BF16 activations"):
        fp8.fp8_linear(torch.zeros(4, 16), torch.zeros(8, 16))
    with pytest.raises(ValueError, match=r"Expected x \[..., K\]"):
        fp8.fp8_linear(torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(8, 24))


def _quantize(**over):
    a = dict(x=P, ldx=64, x_f32=0, rows=4, cols=64, form=3, scale=0, q=P, ldq=64, s=P, ld_s=4, qt=P,
             ldqt=16, st=P, ld_st=4)
    a.update(over)
    _hip.call("ws_fp8_quantize", *a.values(), None)


@pytest.mark.parametrize("over,match", [
    (dict(x=None), "null operand"), (dict(rows=0), "invalid quantization sizes"),
    (dict(ldx=63), "leading dimension"), (dict(x_f32=2), "input type"), (dict(form=5), "form"),
    (dict(scale=2), "scale type"), (dict(q=None), "null output"), (dict(ldq=56), "16 bytes"),
    (dict(q=P + 8), "16-byte"), (dict(ld_s=0), "leading dimension"), (dict(qt=None), "null output"),
    (dict(ldqt=8), "multiple of 16"), (dict(ld_st=0), "leading dimension"),
    (dict(scale=1, ld_s=3), "leading dimension"), (dict(scale=1, ld_st=63), "leading dimension")])
def test_quantization_arguments(over, match):
    with pytest.raises(RuntimeError, match=match):
        _quantize(**over)


def _mm(**over):
    a = dict(a=P, lda=256, sa=P, ld_sa=4, ra=1, b=P, ldb=256, sb=P, ld_sb=4, rb=128, scale=0, c=P,
             ldc=8, m=8, n=8, k=256, ws=None)
    a.update(over)
    _hip.call("ws_fp8_mm", *a.values(), None)


@pytest.mark.parametrize("over,match", [
    (dict(a=None), "null operand"), (dict(m=0), "positive"), (dict(k=8), "16-byte pieces"),
    (dict(lda=240), "16-byte pieces"), (dict(b=P + 4), "16-byte pieces"),
    (dict(lda=1 << 27), "too long"), (dict(scale=7), "scale type"), (dict(ra=64), "1 or 128"),
    (dict(ldc=7), "leading dimension"), (dict(c=P + 1), "misaligned"),
    (dict(ldc=4_200_000), "row stride"), (dict(sa=None), "null scale"), (dict(ld_sa=3), "e8m0"),
    (dict(ld_sb=0), "e8m0"), (dict(scale=1, ld_sa=7), "FP32 scales of A"),
    (dict(scale=1, ld_sa=8, rb=1, ld_sb=10), "FP32 scales of B"),
    (dict(scale=1, ld_sa=8, rb=1, ld_sb=8, sb=P + 4), "FP32 scales of B"),
    (dict(m=64, k=8192, lda=8192, ldb=8192, ld_sa=64, ld_sb=64), "workspace")])
def test_product_arguments(over, match):
    with pytest.raises(RuntimeError, match=match):
        _mm(**over)


def test_pack_arguments():
    with pytest.raises(RuntimeError, match="null operand"):
        _hip.call("ws_fp8_pack", None, 8, 1, P, 16, 4, 8, None)
    with pytest.raises(RuntimeError, match="invalid matrix"):
        _hip.call("ws_fp8_pack", P, 0, 1, P, 16, 4, 8, None)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        _hip.call("ws_fp8_pack", P, 8, 1, P, 24, 4, 8, None)


def test_reference_rounding_is_e4m3():
    """The 64-bit reference rounds as torch's own conversion does, over every pair of
    neighbouring values, their midpoint and either side of it."""
    import numpy as np

    from fp8_reference import e4m3_round

    values = torch.arange(127, dtype=torch.uint8).view(E4M3).double().numpy()  # 0 .. 448
    mid = (values[1:] + values[:-1]) / 2
    x = np.concatenate([values, mid, np.nextafter(mid, 0, dtype=np.float64), mid * (1 + 2e-7)])
    x = np.concatenate([x, -x]).astype(np.float32)
    want = torch.from_numpy(x).to(E4M3).double().numpy()
    np.testing.assert_array_equal(e4m3_round(x.astype(np.float64)), want)


def _plan(m, n, k, rows=128, scale=0):
    import ctypes

    need, splits = ctypes.c_int64(), ctypes.c_int()
    tile = _hip.library().ws_fp8_mm_plan(m, n, k, rows, scale, ctypes.byref(need), ctypes.byref(splits))
    return tile, need.value, splits.value


def test_plans():
    """Few rows take their own kernel, full rounds of 256 x 256 tiles run whole, and tiles that
    would leave compute units idle are split along the reduction, with room for every slice."""
    assert _plan(1, 2048, 5632)[0] == 5 and _plan(32, 2048, 5632)[0] == 5
    assert _plan(8192, 8192, 8192) == (0, 0, 1)
    assert _plan(0, 8, 16)[0] == -1
    for shape in ((64, 2048, 5632), (128, 1280, 4480), (11264, 2048, 16384), (1280, 1280, 16384)):
        tile, need, splits = _plan(*shape)
        assert splits > 1 and need % (4 * splits) == 0 and need > 0, shape
        assert _hip.query("ws_fp8_mm_workspace_bytes", *shape, 128, 0) == need
    # FP32 scales by rows never take the 256 x 256 tile.
    assert all(_plan(m, 8192, 4096, 1, 1)[0] != 0 for m in (512, 4096, 16384))
