"""Static check of private scratch use by the residual norm's, the embedding's and the grouped products'
kernels (CPU only), from the compiler's resource remarks."""
import pytest
from test_kernel_resources import HIPCC, _scratch_by_kernel

pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")


@pytest.mark.parametrize("source,names,most", [
    ("residual_norm.hip", ["add_rmsnorm_kernel", "add_rmsnorm_bwd_kernel"], {}),
    ("embedding.hip", ["embed_lookup_kernel", "embed_sort_kernel", "embed_grad_kernel", "embed_join_kernel"], {}),
    # The input gradients' 256 x 256 tile keeps a few values of its epilogue there.
    ("grouped.hip", ["grouped_fast_kernel", "grouped_ring_kernel", "grouped_grad_fast_kernel",
                     "grouped_grad_ring_kernel", "grouped_few_kernel"], {"grouped_fast_kernelILi1E": 64})])
def test_kernels_use_no_private_scratch(source, names, most, tmp_path):
    scratch = _scratch_by_kernel(source, tmp_path)
    for name in names:
        assert any(name in k for k in scratch), (name, sorted(scratch))
    used = {k: v for k, v in scratch.items() if any(n in k for n in names) and v}
    assert all(any(n in k and v <= limit for n, limit in most.items()) for k, v in used.items()), used
