"""Static check of private scratch use by the smaller kernels beside those of test_layer_resources.py (CPU
only)."""
import pytest
from test_kernel_resources import HIPCC, _scratch_by_kernel

pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")


@pytest.mark.parametrize("source,names", [("embedding.hip", ["embed_few_kernel"]),
                                          ("grouped.hip", ["grouped_join_kernel", "copy_rows_kernel"]),
                                          ("residual_norm.hip", ["rms_weight_reduce_kernel"])])
def test_kernels_use_no_private_scratch(source, names, tmp_path):
    scratch = _scratch_by_kernel(source, tmp_path)
    for name in names:
        found = {k: v for k, v in scratch.items() if name in k}
        assert found and not any(found.values()), (name, found)
