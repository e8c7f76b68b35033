"""The embedding's scale is an FP32 value (GPU)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("scale", [float("inf"), float("nan"), 1e300, -4e38])
def test_scales_that_fp32_does_not_hold_are_refused(scale, native, monkeypatch):
    from ops import _hip
    from ops.embedding_execution import embedding, embedding_accumulate_

    if not native:
        monkeypatch.setattr(_hip, "host_ops", lambda: None)
    tokens, table = torch.arange(3, device="cuda"), torch.ones((5, 16), device="cuda")
    with pytest.raises(ValueError, match="scale must be finite"):
        embedding(tokens, table, scale)
    with pytest.raises(ValueError, match="scale must be finite"):
        embedding_accumulate_(table, tokens, table[:3], scale)
    assert (table == 1).all()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("scale", [3.4e38, -1e-44, 0.0])
def test_the_largest_and_smallest(scale, native, monkeypatch):
    from ops import _hip
    from ops.embedding_execution import embedding

    if not native:
        monkeypatch.setattr(_hip, "host_ops", lambda: None)
    tokens, table = torch.arange(3, device="cuda"), torch.ones((5, 16), device="cuda")
    assert torch.equal(embedding(tokens, table, scale, torch.float32), (table * scale)[:3])
