"""What a recorded grouped product keeps until its backward (GPU): dx needs the weights, dW needs x, and nothing
else is kept or has to stay as it was."""
import weakref

import pytest
import torch

from test_gpu_grouped import BF16, F32, _check, _make, _offsets

pytestmark = pytest.mark.gpu
ROWS, GROUPS = 60, 3


@pytest.fixture(params=[True, False], ids=["native", "python"])
def form(request, monkeypatch):
    from ops import _hip

    if not request.param:
        monkeypatch.setattr(_hip, "host_ops", lambda: None)


def _problem(k, dtype, wants):
    x, w, dy = _make(ROWS, GROUPS, 64, k, dtype, seed=k)
    x.requires_grad_("x" in wants)
    w.requires_grad_("w" in wants)
    return x, w, dy, _offsets(ROWS, GROUPS, "router")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [72, 77])
def test_frozen_weights_do_not_keep_x(k, dtype, form):
    from ops.grouped_execution import grouped_mm

    x, w, dy, offsets = _problem(k, dtype, "x")
    rows = x * 1.0
    kept, before = weakref.ref(rows.untyped_storage()), rows.detach().clone()
    assert kept() is not None
    y = grouped_mm(rows, w, offsets.cuda())
    del rows
    assert kept() is None
    dx, = torch.autograd.grad(y, [x], dy)
    _check(before, w, dy, offsets, y.detach(), dx=dx)


def _storages(call):
    """Data pointers and bytes of the storages that a call saves."""
    saved = {}

    def pack(t):
        s = t.untyped_storage()
        saved[s.data_ptr()] = saved.get(s.data_ptr(), 0) + 1
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        return call(), saved


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [72, 77])
@pytest.mark.parametrize("wants", ["x", "w", "xw"])
def test_saved_tensors(wants, k, dtype, form):
    from ops.grouped_execution import grouped_mm

    x, w, dy, offsets = _problem(k, dtype, wants)
    device_offsets = offsets.cuda()
    y, saved = _storages(lambda: grouped_mm(x, w, device_offsets))
    saved.pop(0, None)  # (tensors without elements)
    copied_x, copied_w = k % 8 != 0, k % 8 != 0 or dtype == F32
    # A copied operand stands for the original, which is not kept beside it.
    assert (x.data_ptr() in saved) == ("w" in wants and not copied_x)
    assert (w.data_ptr() in saved) == ("x" in wants and not copied_w)
    assert len(saved) == 1 + len(wants) and set(saved.values()) == {1}
    assert device_offsets.data_ptr() in saved


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [72, 77])
@pytest.mark.parametrize("wants", ["x", "w"])
def test_the_other_operand_may_change(wants, k, dtype, form):
    from ops.grouped_execution import grouped_mm

    x, w, dy, offsets = _problem(k, dtype, wants)
    x0, w0 = x.detach().clone(), w.detach().clone()
    y = grouped_mm(x, w, offsets.cuda())
    with torch.no_grad():
        (x if wants == "x" else w).fill_(float("nan"))
    got, = torch.autograd.grad(y, [x if wants == "x" else w], dy)
    _check(x0, w0, dy, offsets, y.detach(), **{"d" + wants: got})


@pytest.mark.parametrize("changed", ["x", "w"])
def test_an_operand_that_is_read_may_not_change(changed, form):
    from ops.grouped_execution import grouped_mm

    x, w, dy, offsets = _problem(72, BF16, "xw")
    y = grouped_mm(x, w, offsets.cuda())
    with torch.no_grad():
        (x if changed == "x" else w).mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x, w], dy)


@pytest.mark.parametrize("interior", [False, True])
@pytest.mark.parametrize("wants", ["x", "w", "xw"])
def test_second_derivatives_stay_refused(wants, interior, form):
    """To every input that the call recorded, leaves or not, also those that a gradient does not depend on."""
    from ops.grouped_execution import grouped_mm

    x, w, dy, offsets = _problem(72, BF16, wants)
    a, b = (x * 1.0, w * 1.0) if interior else (x, w)
    leaves = [t for t, name in ((x, "x"), (w, "w")) if name in wants]
    first = torch.autograd.grad(grouped_mm(a, b, offsets.cuda()), leaves, dy, create_graph=True)
    for g in first:
        for leaf in leaves:
            with pytest.raises(RuntimeError, match="twice"):
                torch.autograd.grad(g.float().sum(), [leaf], retain_graph=True, allow_unused=True)


def test_recomputed(form):
    """Under checkpointing, whose second forward has to keep the same tensors."""
    from torch.utils.checkpoint import checkpoint

    from ops.grouped_execution import grouped_mm

    for wants, k, dtype in (("x", 72, BF16), ("w", 77, F32), ("xw", 77, BF16)):
        x, w, dy, offsets = _problem(k, dtype, wants)
        leaves = [t for t, name in ((x, "x"), (w, "w")) if name in wants]
        offsets = offsets.cuda()
        want = torch.autograd.grad(grouped_mm(x, w, offsets), leaves, dy)
        got = torch.autograd.grad(checkpoint(grouped_mm, x, w, offsets, use_reentrant=False), leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_compiled_backward():
    """The backward itself compiled."""
    from torch._dynamo import compiled_autograd

    from ops.grouped_execution import grouped_mm

    x, w, dy, offsets = _problem(72, F32, "xw")
    offsets = offsets.cuda()
    grouped_mm(x, w, offsets).backward(dy)
    want = [x.grad.clone(), w.grad.clone()]
    x.grad = w.grad = None
    with compiled_autograd._enable(torch.compile(backend="aot_eager")):
        grouped_mm(x, w, offsets).backward(dy)
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
