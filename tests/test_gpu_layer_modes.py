"""The residual norm, the embedding and the grouped products under PyTorch's other modes: forward-mode
tensors, functorch's derivatives and a second differentiation are refused, vmap and fake tensors reach
the operators, and compiled functions hold them whole (GPU)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _calls():
    from ops.embedding_execution import embedding
    from ops.grouped_execution import grouped_mm
    from ops.residual_norm import add_rmsnorm, rmsnorm_quantize

    g = torch.Generator().manual_seed(1)
    make = lambda *s: torch.randn(s, generator=g).to(BF16).cuda()
    x, residual, weight = make(5, 64), make(5, 64), make(64).float()
    table, experts = make(30, 64), make(3, 48, 64)
    tokens = torch.tensor([3, 1, 4, 1, 5]).cuda()
    offsets = torch.tensor([0, 2, 2, 5]).cuda()
    return {"norm": (lambda t: add_rmsnorm(t, residual, weight)[0], x),
            "norm residual": (lambda t: add_rmsnorm(x, t, weight)[1], residual),
            "norm weight": (lambda t: add_rmsnorm(x, residual, t)[0], weight),
            "embedding": (lambda t: embedding(tokens, t, 0.5), table),
            "experts": (lambda t: grouped_mm(t, experts, offsets), x),
            "experts weight": (lambda t: grouped_mm(x, t, offsets), experts),
            "quantize": (lambda t: rmsnorm_quantize(t, weight, residual=residual)[2], x)}


NAMES = ["norm", "norm residual", "norm weight", "embedding", "experts", "experts weight"]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("requires", [False, True])
@pytest.mark.parametrize("name", [*NAMES, "quantize"])
def test_forward_mode_is_refused(name, requires, native, monkeypatch):
    """A tangent is never dropped."""
    from ops import _hip

    call, x = _calls()[name]
    if not native:
        monkeypatch.setattr(_hip, "host_ops", lambda: None)
    with fwd.dual_level():
        dual = fwd.make_dual(x.requires_grad_(requires), torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            call(dual)
    assert call(x).shape[0] == 5  # the same without a tangent


@pytest.mark.parametrize("name", NAMES)
def test_functorch_derivatives_are_refused(name):
    call, x = _calls()[name]
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: call(t).float().sum())(x)


@pytest.mark.parametrize("name", NAMES)
def test_vmap(name):
    call, x = _calls()[name]
    many = torch.stack([x, x * 0.5, x + 1.0])
    assert torch.equal(torch.func.vmap(call)(many), torch.stack([call(t) for t in many]))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", ["norm", "norm weight", "embedding", "experts", "experts weight"])
def test_recorded_backward(name, native, monkeypatch):
    """create_graph gives the plain first derivative; the second is refused."""
    from ops import _hip

    if not native:
        monkeypatch.setattr(_hip, "host_ops", lambda: None)
    call, x = _calls()[name]
    leaf = x.clone().requires_grad_(True)
    out = call(leaf).float()
    up = torch.linspace(-1, 1, out.numel()).view(out.shape).cuda().requires_grad_(True)
    want, = torch.autograd.grad((out * up.detach()).sum(), [leaf], retain_graph=True)
    got, = torch.autograd.grad((out * up).sum(), [leaf], create_graph=True)
    assert torch.equal(got, want)
    if name != "embedding":  # whose gradient does not depend on the table
        with pytest.raises(RuntimeError, match="twice"):
            torch.autograd.grad(got.float().sum(), [leaf], allow_unused=True)
    got, = torch.autograd.grad((call(leaf).float() * up).sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(got.float().sum(), [up], allow_unused=True)


@pytest.mark.parametrize("name", NAMES)
def test_compiled_whole(name):
    """fullgraph: the operators are in the graph, with their gradients."""
    call, x = _calls()[name]
    got, want = [], []
    for f, out in ((torch.compile(call, fullgraph=True, backend="aot_eager"), got), (call, want)):
        leaf = x.clone().requires_grad_(True)
        y = f(leaf)
        out += [y, torch.autograd.grad(y.float().sum(), [leaf])[0]]
        with torch.no_grad():
            out.append(f(x))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("stream", [True, False])
def test_compiled_quantization(stream, native, monkeypatch):
    """The 8-bit norm and the product that reads it in one compiled function; without the C++
    operators they run eagerly in it, as do the others."""
    from ops import _hip
    from ops import fp8_execution as fp8
    from ops.embedding_execution import embedding, embedding_accumulate_
    from ops.grouped_execution import grouped_mm
    from ops.residual_norm import add_rmsnorm, rmsnorm_quantize

    if not native:
        monkeypatch.setattr(_hip, "host_ops", lambda: None)
    g = torch.Generator().manual_seed(4)
    x, residual = (torch.randn((7, 200), generator=g).to(BF16).cuda() for _ in range(2))
    weight, experts = torch.ones(200, device="cuda"), torch.randn((2, 200, 200), generator=g).to(BF16).cuda()
    tokens, offsets = torch.arange(7, device="cuda"), torch.tensor([0, 3, 7], device="cuda")

    def step(x):
        q, scale, out = rmsnorm_quantize(x, weight, residual=residual if stream else None)
        q32, scale32, _ = rmsnorm_quantize(x, weight, scale_dtype=F32)
        y, _ = add_rmsnorm(x + embedding(tokens, residual), residual, weight)
        grad = embedding_accumulate_(torch.zeros((9, 200), device="cuda"), tokens, y)
        return (q.float(), scale.view(torch.uint8), out * 2, q32.float(), scale32 * 1, grad,
                grouped_mm(y, experts, offsets))

    want = step(x)
    got = torch.compile(step, backend="aot_eager")(x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert [t.stride() for t in got[:2]] == [t.stride() for t in want[:2]]


@pytest.mark.parametrize("odd", [False, True])
def test_compiled_with_any_row_count(odd):
    """One compiled function for all numbers of rows."""
    from ops.embedding_execution import embedding
    from ops.grouped_execution import grouped_mm
    from ops.residual_norm import add_rmsnorm

    g = torch.Generator().manual_seed(2)
    d, n = (37, 11) if odd else (64, 48)
    leaf = lambda *s: torch.randn(s, generator=g).cuda().requires_grad_(True)
    table, weight, experts = leaf(30, d), leaf(d), leaf(3, n, d)

    def step(tokens, offsets):
        h = embedding(tokens, table, 0.5)
        y, stream = add_rmsnorm(h, h.float(), weight)
        return grouped_mm(y, experts, offsets), stream

    compiled = torch.compile(step, fullgraph=True, backend="aot_eager", dynamic=True)
    for rows in (5, 12, 700):
        tokens = torch.randint(0, 30, (rows,), generator=g).cuda()
        offsets = torch.tensor([0, rows // 3, rows // 2, rows]).cuda()
        got, want = compiled(tokens, offsets), step(tokens, offsets)
        up = [torch.ones_like(t) for t in want]
        got = [*got, *torch.autograd.grad(got, [table, weight, experts], up)]
        want = [*want, *torch.autograd.grad(want, [table, weight, experts], up)]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rows


def test_inference_mode():
    from ops.embedding_execution import embedding_accumulate_

    for name, (call, x) in _calls().items():
        want = call(x)
        with torch.inference_mode():
            assert torch.equal(call(x), want), name
    with torch.inference_mode():
        grad = torch.zeros((30, 8), device="cuda")
        tokens, dy = torch.tensor([3, 3], device="cuda"), torch.ones((2, 8), device="cuda")
        assert (embedding_accumulate_(grad, tokens, dy)[3] == 2).all()


@pytest.mark.parametrize("requires", [False, True])
def test_fake_tensors(requires):
    """Shapes and types without data."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from ops.embedding_execution import embedding
    from ops.grouped_execution import grouped_mm
    from ops.residual_norm import add_rmsnorm

    with FakeTensorMode():
        make = lambda *s, dtype=BF16: torch.empty(s, dtype=dtype, device="cuda", requires_grad=requires)
        x, residual, weight = make(7, 40), make(7, 40, dtype=F32), make(40, dtype=F32)
        table, experts = make(90, 40, dtype=F32), make(3, 13, 40, dtype=F32)
        tokens = torch.zeros(7, dtype=torch.int64, device="cuda")
        y, stream = add_rmsnorm(x, residual, weight)
        e = embedding(tokens, table)
        z = grouped_mm(x, experts, torch.zeros(4, dtype=torch.int64, device="cuda"))
        assert [(tuple(t.shape), t.dtype) for t in (y, stream, e, z)] == [
            ((7, 40), BF16), ((7, 40), F32), ((7, 40), BF16), ((7, 13), BF16)]
        if requires:
            leaves = [x, residual, weight, table, experts]
            grads = torch.autograd.grad((y.float().sum() + stream.sum() + e.float().sum() + z.float().sum()), leaves)
            assert [(g.shape, g.dtype) for g in grads] == [(t.shape, t.dtype) for t in leaves]


def test_saved_stream_that_was_changed_is_refused():
    """The backward reads the returned stream; one that was written to in place is not used."""
    from ops.residual_norm import add_rmsnorm

    x = torch.randn((4, 64), device="cuda").to(BF16).requires_grad_(True)
    y, stream = add_rmsnorm(x, x.detach(), torch.ones(64, device="cuda"))
    with torch.no_grad():
        stream.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()
