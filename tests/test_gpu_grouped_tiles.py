"""Grouped products on the tiles, and loops over tiles, that the other tests' sizes do not choose (GPU)."""
import pytest
import torch

from test_gpu_grouped import BF16, F32, F64, GRAD, NN, NT, SIZES, _check, _close, _make, _offsets

pytestmark = pytest.mark.gpu

# Rows, groups, n, k whose weight gradients take one 128 x 128 workgroup on a compute unit, and two.
ALONE = [(2048, 2, 1024, 2048), (4096, 4, 1024, 1024)]
PAIRS = [(20, 8, 1288, 2056), (4096, 64, 512, 1280)]


def _tile(*args):
    from ops import _hip

    return _hip.query("ws_grouped_tile", *args)


@pytest.mark.parametrize("kind", ["router", "one", "gaps", "even"])
@pytest.mark.parametrize("tile,sizes,dtype", [(2, s, t) for s in ALONE for t in (BF16, F32)] + [(1, s, F32) for s in PAIRS])
def test_weight_gradients_of_128_rows(tile, sizes, dtype, kind):
    from ops.grouped_execution import grouped_mm

    rows, groups, n, k = sizes
    assert _tile(*sizes, GRAD) == tile
    x, w, dy = _make(rows, groups, n, k, dtype, seed=k)
    offsets = _offsets(rows, groups, kind, seed=n)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = grouped_mm(x, w, offsets.cuda())
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert dw.dtype == dtype
    _check(x.detach(), w, dy, offsets, y, dx, dw)


def test_every_gradient_tile_is_reached():
    assert {_tile(r, g, n, k, GRAD) for r, g, n, k in SIZES + ALONE} == {0, 1, 2, 3, 4}


ROWS_OF, COLS_OF = {1: 128, 2: 128, 3: 64, 4: 64, 5: 16}, {1: 128, 2: 128, 3: 128, 4: 64, 5: 32}


# Sizes of which a workgroup takes several tiles, by the tile that they choose: rows, groups, columns, reduction.
@pytest.mark.parametrize("kind", ["router", "gaps"])
@pytest.mark.parametrize("form,tile,rows,groups,cols,depth", [
    (NT, 1, 102489, 1297, 64, 8), (NT, 2, 276893, 90, 72, 72), (NT, 3, 6019, 951, 144, 8), (NT, 4, 12284, 1877, 16, 8),
    (NT, 5, 1956, 1959, 16, 8), (NN, 1, 102489, 1297, 64, 8), (NN, 2, 232728, 447, 72, 80), (NN, 3, 2914, 2005, 72, 8),
    (NN, 4, 2429, 2090, 16, 8)])
def test_several_tiles_of_a_workgroup(form, tile, rows, groups, cols, depth, kind):
    from ops.grouped_execution import grouped_mm

    assert _tile(rows, groups, cols, depth, form) == tile
    tiles = (rows // ROWS_OF[tile] + min(groups + 2, rows)) * -(-cols // COLS_OF[tile])
    assert tiles // (4 * torch.cuda.get_device_properties(0).multi_processor_count) >= 2
    n, k = (cols, depth) if form == NT else (depth, cols)
    x, w, dy = _make(rows, groups, n, k, seed=rows)
    offsets = _offsets(rows, groups, kind, seed=n)
    owner = torch.bucketize(torch.arange(rows), offsets, right=True) - 1  # -1 or groups: none
    known = ((owner >= 0) & (owner < groups)).cuda()
    owner = owner.clamp(0, groups - 1).cuda()
    x.requires_grad_(form == NN)
    got = grouped_mm(x, w, offsets.cuda())
    if form == NN:
        got, = torch.autograd.grad(got, x, dy)
    for part in torch.arange(rows, device="cuda").split(16384):
        mine = w[owner[part]].to(F64) * known[part][:, None, None]
        a = (x.detach()[part].to(F64)[:, None] if form == NT else dy[part].to(F64)[:, :, None]) * mine
        over = 2 if form == NT else 1
        _close(got[part], a.sum(over), a.abs().sum(over), depth)
