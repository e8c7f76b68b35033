"""Static check of private scratch use by the 8-bit and token-score kernels (CPU only).

Their register budgets are what their schedules are built on (two waves on a SIMD for the 256 x
256 product, eight workgroups on a compute unit for the rows of logits): a spill would go
unnoticed by every other test. The compiler's resource remarks, built with the library's flags,
give each kernel's scratch bytes per lane.
"""
import pytest
from test_kernel_resources import HIPCC, _scratch_by_kernel

pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")


@pytest.mark.parametrize("source,names", [
    ("fp8.hip", ["quantize_kernel", "pack_bytes_kernel", "gemm_fp8_kernel", "gemm_fp8_ring_kernel",
                 "gemm_fp8_skinny_kernel", "fp8_join_kernel"]),
    ("scores.hip", ["score_rows_kernel", "score_join_kernel", "score_grad_kernel",
                    "score_coef_kernel", "FEpiScoreStats", "FEpiScoreGrad"])])
def test_kernels_use_no_private_scratch(source, names, tmp_path):
    scratch = _scratch_by_kernel(source, tmp_path)
    for name in names:
        assert any(name in k for k in scratch), (name, sorted(scratch))
    assert {k: v for k, v in scratch.items() if v} == {}
