"""The 8-bit residual norm whole in compiled functions, as the other operators (GPU)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
E8M0 = torch.float8_e8m0fnu


@pytest.fixture(autouse=True)
def fresh():
    """(Every case compiles the same functions; their number is limited.)"""
    torch._dynamo.reset()
    yield
    torch._dynamo.reset()


def _bytes(outputs):
    return [t.contiguous().view(torch.uint8) for t in outputs]


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("scale_dtype", [E8M0, F32])
@pytest.mark.parametrize("stream", [None, BF16, F32])
@pytest.mark.parametrize("d", [200, 1280])
def test_fullgraph(d, stream, scale_dtype, dynamic):
    from ops.residual_norm import rmsnorm_quantize

    weight = torch.linspace(0.5, 1.5, d, device="cuda")

    def step(x, residual):
        q, scale, out = rmsnorm_quantize(x * 2, weight, residual=residual, scale_dtype=scale_dtype)
        return q, scale, out + 1

    compiled = torch.compile(step, fullgraph=True, backend="aot_eager", dynamic=dynamic)
    g = torch.Generator().manual_seed(d)
    for rows in (7, 12, 700) if dynamic else (7,):
        x = torch.randn((rows, d), generator=g).to(BF16).cuda()
        residual = None if stream is None else torch.randn((rows, d), generator=g).to(stream).cuda()
        got, want = compiled(x, residual), step(x, residual)
        assert [(t.shape, t.dtype, t.stride()) for t in got] == [(t.shape, t.dtype, t.stride()) for t in want]
        assert all(torch.equal(a, b) for a, b in zip(_bytes(got), _bytes(want)))
