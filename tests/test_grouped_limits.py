"""How many tiles grouped products take, one size on each side (CPU; the queries answer for 256 compute units where
there is no GPU)."""
import pytest

from ops import _hip

NT, NN, GRAD = 0, 1, 2


def _tile(*args):
    return _hip.query("ws_grouped_tile", *args)


# 16384 rows in 16384 groups: 16448 tiles of 256 rows at most, 1020 times which is below 2^24.
@pytest.mark.parametrize("form", [NT, NN])
@pytest.mark.parametrize("n,fits", [(16, True), (11264, True), (261120, True), (261121, False)])
def test_products(n, fits, form):
    assert (_tile(16384, 16384, n, 16, form) >= 0) == fits


def test_tiles_give_way_to_larger_ones():
    """Where a kernel's tiles are too many, a larger tile takes the product."""
    few, other = _tile(16384, 16384, 11264, 16, NT), _tile(16384, 16384, 32768, 16, NT)
    assert few == 5 and 0 <= other < 5
    # One row a group and a long reduction: 16 columns, while they need no more than a workgroup each.
    assert _tile(4096, 4096, 4096, 2048, NT) == 6 and _tile(4096, 4096, 32768, 2048, NT) == 5


# Tiles of 256 x 256: 16384 times 255, and times 256.
@pytest.mark.parametrize("n,k,fits", [(8, 32904, True), (3840, 4352, True), (4096, 4096, False), (4352, 3840, True),
                                      (256, 65536, False)])
def test_weight_gradients(n, k, fits):
    assert (_tile(17, 16384, n, k, GRAD) >= 0) == fits
    if not fits:
        with pytest.raises(RuntimeError, match="tiles"):
            _hip.call("ws_grouped_backward_check", 17, 16384, n, k, 0, 1, 0)
    else:
        _hip.call("ws_grouped_backward_check", 17, 16384, n, k, 1, 1, 1)
    _hip.call("ws_grouped_backward_check", 17, 16384, n, k, 1, 0, 0)


@pytest.mark.parametrize("args,match", [
    ((4, 0, 8, 8, 1, 1, 0), "groups"), ((-1, 2, 8, 8, 1, 1, 0), "shape"),
    ((16384, 16384, 8, 261121, 1, 0, 0), "tiles"), ((4, 2, 8, 2200000, 1, 1, 1), "stride"),
    ((4, 2, 4200000, 8, 1, 0, 0), "stride"), ((4, 2, 8, 4200000, 0, 1, 0), "stride")])
def test_backward_check(args, match):
    with pytest.raises(RuntimeError, match=match):
        _hip.call("ws_grouped_backward_check", *args)


@pytest.mark.parametrize("args", [(0, 2, 8, 8, 1, 1, 0), (4, 2, 8, 2200000, 1, 1, 0), (4, 2, 8, 2200000, 1, 0, 1),
                                  (16384, 16384, 261121, 8, 1, 0, 0), (1, 1, 1, 1, 1, 1, 1)])
def test_backward_check_passes(args):
    _hip.call("ws_grouped_backward_check", *args)
