"""Grouped products of very many tiles (GPU): every call that is recorded has its gradients, and more tiles than
one launch takes workgroups are shared by fewer of them."""
import pytest
import torch

from test_gpu_grouped import BF16, F32, F64, NT, _close

pytestmark = pytest.mark.gpu


def test_more_tiles_than_workgroups():
    """6 million tiles of a short reduction, sixteen a workgroup."""
    from ops import _hip
    from ops.grouped_execution import grouped_mm

    rows = groups = 16384
    n, k = 11264, 16
    assert _hip.query("ws_grouped_tile", rows, groups, n, k, NT) == 5
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn((rows, k), generator=g, device="cuda", dtype=BF16)
    w = torch.randn((groups, n, k), generator=g, device="cuda", dtype=BF16)
    lengths = torch.ones(groups, dtype=torch.int64)
    lengths[5], lengths[6], lengths[-1] = 0, 2, 0  # one group of two rows, and one row behind the last
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)])
    owner = torch.repeat_interleave(torch.arange(groups), lengths)
    with torch.no_grad():
        y = grouped_mm(x, w, offsets.cuda())
    assert not y[len(owner):].any()
    for part in torch.arange(len(owner)).split(1024):
        a, b = x[part].to(F64)[:, None], w[owner[part]].to(F64)
        _close(y[part], (a * b).sum(2), (a * b).abs().sum(2), k)


def test_more_tiles_than_workgroups_of_a_long_reduction():
    """4.5 million tiles, two a workgroup; the weight is shared by all groups."""
    from ops import _hip
    from ops.grouped_execution import grouped_mm

    rows = groups = 4096
    n, k = 32768, 264
    assert _hip.query("ws_grouped_tile", rows, groups, n, k, NT) == 5
    g = torch.Generator("cuda").manual_seed(2)
    x = torch.randn((rows, k), generator=g, device="cuda", dtype=BF16)
    w = torch.randn((1, n, k), generator=g, device="cuda", dtype=BF16)
    with torch.no_grad():
        y = grouped_mm(x, w.expand(groups, n, k), torch.arange(groups + 1, device="cuda"))
    for part in torch.arange(rows).split(512):
        a, b = x[part].to(F64), w[0].to(F64)
        _close(y[part], a @ b.T, a.abs() @ b.abs().T, k)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradient_of_many_narrow_weights(dtype):
    """Of whose tiles only the largest are few enough."""
    from ops import _hip
    from ops.grouped_execution import grouped_mm

    rows, groups, n, k = 17, 16384, 8, 32904
    assert _hip.query("ws_grouped_tile", rows, groups, n, k, 2) == 0
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn((rows, k), generator=g, device="cuda", dtype=BF16).requires_grad_(True)
    w = torch.randn((groups, n, k), generator=g, device="cuda", dtype=BF16).to(dtype).requires_grad_(True)
    dy = torch.randn((rows, n), generator=g, device="cuda", dtype=BF16)
    owner = torch.tensor([0, 0, 0, 7, 7, 100, 8191, 8192, 8192, 9000, 9001, 9002, 16000, 16381, 16381, 16383, 16383])
    offsets = torch.searchsorted(owner, torch.arange(groups + 1))
    y = grouped_mm(x, w, offsets.cuda())
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    empty = torch.ones(groups, dtype=torch.bool)
    for e in owner.unique().tolist():
        empty[e] = False
        lo, hi = offsets[e], offsets[e + 1]
        a, b, d = x.detach()[lo:hi].to(F64), w.detach()[e].to(BF16).to(F64), dy[lo:hi].to(F64)
        _close(y[lo:hi], a @ b.T, a.abs() @ b.abs().T, k)
        _close(dx[lo:hi], d @ b, d.abs() @ b.abs(), n)
        _close(dw[e], d.T @ a, d.abs().T @ a.abs(), int(hi - lo))
    seen = dw.view(groups, -1).count_nonzero(1).cpu()
    assert not seen[empty].any() and seen[~empty].all()


@pytest.mark.parametrize("native", [True, False])
def test_a_gradient_that_does_not_fit_is_refused_at_once(native, monkeypatch):
    from ops import _hip
    from ops.grouped_execution import grouped_mm

    if not native:
        monkeypatch.setattr(_hip, "host_ops", lambda: None)
    groups, n = 16384, 4096
    x = torch.ones((4, n), device="cuda", dtype=BF16)
    leaf = torch.ones((1, n, n), device="cuda", dtype=BF16).requires_grad_(True)
    offsets = torch.arange(groups + 1, device="cuda").clamp(max=4)
    with pytest.raises(RuntimeError, match="tiles"):
        grouped_mm(x, leaf.expand(groups, n, n), offsets)
    if native:  # (without gradients the weights are read where they lie)
        with torch.no_grad():
            assert (grouped_mm(x, leaf.expand(groups, n, n), offsets) == n).all()


def test_copies_of_very_many_rows():
    """67 million rows of a width that is padded, and of a gradient that is cut off again."""
    from ops.grouped_execution import grouped_mm

    rows, groups, n, k = 100, 16384, 4100, 3
    g = torch.Generator("cuda").manual_seed(4)
    x = torch.randn((rows, k), generator=g, device="cuda", dtype=BF16)
    w = torch.randn((groups, n, k), generator=g, device="cuda").requires_grad_(True)
    dy = torch.randn((rows, n), generator=g, device="cuda", dtype=BF16)
    owner = torch.arange(rows) // 2 * 334
    owner[-2:] = groups - 1
    y = grouped_mm(x, w, torch.searchsorted(owner, torch.arange(groups + 1)).cuda())
    dw, = torch.autograd.grad(y, w, dy)
    seen = dw.view(groups, -1).count_nonzero(1).cpu()
    seen[owner] = 0
    assert not seen.any()
    for lo in range(0, rows, 2):
        a, b, d = x[lo:lo + 2].to(F64), w.detach()[owner[lo]].to(BF16).to(F64), dy[lo:lo + 2].to(F64)
        _close(y[lo:lo + 2], a @ b.T, a.abs() @ b.abs().T, k)
        _close(dw[owner[lo]], d.T @ a, d.abs().T @ a.abs(), 2)
