"""Scales that are no matrices are refused alike with and without ``out`` (GPU)."""
import pytest
import torch

from fp8_reference import E8M0, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale_dtype", [E8M0, F32])
@pytest.mark.parametrize("with_out", [False, True])
def test_scales_that_are_no_matrices(with_out, scale_dtype):
    from ops import fp8_execution as fp8

    a, sa = fp8.quantize_rows(torch.randn((20, 256), device="cuda"), scale_dtype)
    b, sb = fp8.quantize_weight(torch.randn((40, 256), device="cuda"), scale_dtype)[:2]
    out = torch.empty((20, 40), dtype=torch.bfloat16, device="cuda") if with_out else None
    for args in ((a, sa, b, sb[0, 0]), (a, sa, b, sb[0]), (a, sa[0, 0], b, sb), (a, sa[:, 0], b, sb)):
        with pytest.raises(ValueError, match="matrix of"):
            fp8.fp8_mm(*args, out=out)
