"""The 8-bit projection and the token scores under PyTorch's other modes: forward-mode tensors and
functorch's derivatives are refused, vmap and fake tensors reach the operators, a recorded backward
gives the first derivative (GPU)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _calls():
    from ops import fp8_execution as fp8
    from ops import token_scores as ts

    g = torch.Generator().manual_seed(1)
    make = lambda *s: torch.randn(s, generator=g).to(BF16).cuda()
    tokens = torch.tensor([3, 1, 4, 1, 5]).cuda()
    weight, head = make(48, 64), make(300, 64)
    return {"scores": (lambda x: ts.token_scores(x, tokens)[0], make(5, 300)),
            "head": (lambda x: ts.linear_token_scores(x, head, tokens)[0], make(5, 64)),
            "head weight": (lambda w: ts.linear_token_scores(head[:5], w, tokens)[0], make(300, 64)),
            "projection": (lambda x: fp8.fp8_linear(x, weight), make(5, 64)),
            "projection weight": (lambda w: fp8.fp8_linear(weight[:5], w), make(48, 64))}


NAMES = ["scores", "head", "head weight", "projection", "projection weight"]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("requires", [False, True])
@pytest.mark.parametrize("name", NAMES)
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
    """(NotImplementedError is a RuntimeError; PyTorch's own refusal of C++ nodes is one too.)"""
    call, x = _calls()[name]
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: call(t).float().sum())(x)


@pytest.mark.parametrize("name", ["scores", "projection"])
def test_vmap(name):
    call, x = _calls()[name]
    many = torch.stack([x, x * 0.5, x + 1.0])
    want = torch.stack([call(t) for t in many])
    assert torch.equal(torch.func.vmap(call)(many), want)


@pytest.mark.parametrize("name", NAMES)
def test_recorded_backward(name):
    """create_graph gives the plain first derivative; the second is refused."""
    call, x = _calls()[name]
    leaf = x.clone().requires_grad_(True)
    out = call(leaf).float()
    up = torch.linspace(-1, 1, out.numel()).view(out.shape).cuda().requires_grad_(True)
    want, = torch.autograd.grad((out * up.detach()).sum(), [leaf], retain_graph=True)
    got, = torch.autograd.grad((out * up).sum(), [leaf], create_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(got.float().sum(), [leaf])
    with pytest.raises(RuntimeError):
        got, = torch.autograd.grad((call(leaf).float() * up).sum(), [leaf], create_graph=True)
        torch.autograd.grad(got.float().sum(), [up])


@pytest.mark.parametrize("requires", [False, True])
def test_fake_logits(requires):
    """Shapes and types of the scores and their gradient, without data."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from ops import token_scores as ts

    with FakeTensorMode():
        x = torch.empty((7, 300), dtype=BF16, device="cuda", requires_grad=requires)
        got = ts.token_scores(x, torch.zeros(7, dtype=torch.int64, device="cuda"), 3)
        assert [(tuple(t.shape), t.dtype) for t in got] == [((7,), F32), ((7,), F32), ((7, 3), F32),
                                                             ((7, 3), torch.int64)]
        assert got.logprob.requires_grad == requires
        if requires:
            dx, = torch.autograd.grad(got.logprob.sum() + got.entropy.sum(), [x])
            assert dx.shape == x.shape and dx.dtype == BF16
