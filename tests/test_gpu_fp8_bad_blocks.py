"""A block that holds an infinity or a NaN is NaN throughout, in every form and in the product."""
import numpy as np
import pytest
import torch

from fp8_reference import BLOCK, E8M0, F32, dequantize, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale_dtype", [E8M0, F32])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_all_of_a_bad_block_is_nan(bad, scale_dtype):
    from ops import fp8_execution as fp8

    x = torch.randn((260, 300), generator=torch.Generator().manual_seed(1)).cuda()
    x[130, 140] = bad
    q, scale, qt, scale_t = (values(t) for t in fp8.quantize_rows_and_columns(x, scale_dtype))
    w, w_scale, wt, wt_scale = (values(t) for t in fp8.quantize_weight(x, scale_dtype))
    with np.errstate(invalid="ignore"):
        for got, rows, cols in ((dequantize(q, scale), slice(130, 131), slice(128, 256)),
                                (dequantize(qt, scale_t).T, slice(128, 256), slice(140, 141)),
                                (dequantize(w, w_scale), slice(128, 256), slice(128, 256)),
                                (dequantize(wt, wt_scale).T, slice(128, 256), slice(128, 256))):
            want = np.zeros_like(got, bool)
            want[rows, cols] = True
            np.testing.assert_array_equal(np.isnan(got), want)
    a = torch.randn((40, 300), generator=torch.Generator().manual_seed(2)).cuda()
    out = fp8.fp8_mm(*fp8.quantize_rows(a, scale_dtype), *fp8.quantize_weight(x, scale_dtype)[:2])
    bad_columns = torch.isnan(out)
    assert bool(bad_columns[:, BLOCK:2 * BLOCK].all())
    assert not bool(bad_columns[:, :BLOCK].any()) and not bool(bad_columns[:, 2 * BLOCK:].any())
