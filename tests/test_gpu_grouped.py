"""Products grouped by expert against plain products of each group in 64 bits (GPU).

Bounds: half a step of the result's type, and FP32 sums of n products (n 2^-24 of their
magnitudes)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24
NT, NN, GRAD = 0, 1, 2


def _offsets(rows, groups, kind, seed=0):
    """Counts of a kind; "gaps" leaves rows before the first group and behind the last."""
    g = torch.Generator().manual_seed(seed)
    if kind == "one":  # all rows in one group
        counts = torch.zeros(groups, dtype=torch.int64)
        counts[groups // 2] = rows
    elif kind == "even":
        counts = torch.full((groups,), rows // groups)
        counts[:rows % groups] += 1
    else:  # like a router's, with empty groups
        liking = torch.randn(groups, generator=g).exp()
        liking[torch.rand(groups, generator=g) < 0.25] = 0
        liking[groups - 1] = 1
        picks = torch.multinomial(liking, max(rows, 1), replacement=True, generator=g)[:rows]
        counts = torch.bincount(picks, minlength=groups)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    if kind == "gaps":
        offsets = offsets.clamp(rows // 7, rows - rows // 5)
    return offsets


def _make(rows, groups, n, k, dtype=BF16, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn((rows, k), generator=g, device="cuda").to(BF16)
    w = (0.05 * torch.randn((groups, n, k), generator=g, device="cuda")).to(dtype)
    dy = torch.randn((rows, n), generator=g, device="cuda").to(BF16)
    return x, w, dy


def _close(got, want, size, terms):
    bound = want.abs() * torch.finfo(got.dtype).eps / 2 + size * terms * U
    off = (got.to(F64) - want).abs()
    assert got.isfinite().all() and (off <= bound).all(), (off / bound.clamp_min(1e-300)).max().item()


def _check(x, w, dy, offsets, y, dx=None, dw=None):
    bounds = offsets.tolist()
    n, k = w.shape[1:]
    seen = torch.zeros(len(x), dtype=torch.bool)
    for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        seen[lo:hi] = True
        a, b = x[lo:hi].to(F64), w[e].detach().to(BF16).to(F64)
        _close(y[lo:hi], a @ b.T, a.abs() @ b.abs().T, k)
        if dx is not None:
            g = dy[lo:hi].to(F64)
            _close(dx[lo:hi], g @ b, g.abs() @ b.abs(), n)
        if dw is not None:
            g = dy[lo:hi].to(F64)
            _close(dw[e], g.T @ a, g.abs().T @ a.abs(), max(1, hi - lo))
    for t in (y, dx):
        if t is not None:
            assert not t[~seen.cuda()].any()


# Rows, groups, n, k. The last five reach the pieces of a last round of 256 x 256 tiles (no whole
# round before it, one, and a last round that is long enough to stay whole).
SIZES = [(1, 1, 8, 8), (1, 5, 64, 72), (7, 3, 16, 200), (16, 64, 96, 264), (20, 8, 1288, 2056), (40, 8, 1288, 264),
         (100, 8, 520, 264), (300, 16, 2056, 136), (100, 9, 264, 1000), (200, 8, 520, 96),
         (300, 4, 512, 512), (700, 70, 64, 64), (1000, 130, 128, 136), (1000, 5, 256, 128), (3000, 3, 2048, 512),
         (4096, 8, 1288, 1280), (4096, 64, 512, 1280), (6000, 32, 1280, 896), (8192, 4, 1280, 520),
         (2600, 2, 2056, 1544), (9000, 4, 2304, 1608), (9000, 4, 1608, 2304), (12000, 3, 2304, 1536),
         (16000, 6, 2048, 1032)]


@pytest.mark.parametrize("kind", ["router", "one", "gaps", "even"])
@pytest.mark.parametrize("sizes", SIZES)
def test_forward_and_backward(sizes, kind):
    from ops.grouped_execution import grouped_mm

    rows, groups, n, k = sizes
    dtype = F32 if (rows + groups) % 2 else BF16
    x, w, dy = _make(rows, groups, n, k, dtype, seed=rows)
    offsets = _offsets(rows, groups, kind, seed=n)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = grouped_mm(x, w, offsets.cuda())
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert y.dtype == dx.dtype == BF16 and dw.dtype == dtype
    _check(x.detach(), w, dy, offsets, y, dx, dw)
    with torch.no_grad():
        assert torch.equal(grouped_mm(x, w, offsets.cuda()), y)


@pytest.mark.parametrize("sizes", [(900, 4500, 24, 40), (600, 300, 200, 136), (5000, 200, 72, 520), (2000, 1500, 264, 40),
                                   (7001, 400, 520, 72), (3000, 64, 2056, 24), (20000, 4, 40, 264),
                                   (16384, 16384, 16, 64)])
def test_many_groups(sizes):
    """More groups than lanes, and more than 64 on a lane; short reductions, of which a workgroup takes
    several tiles."""
    from ops.grouped_execution import grouped_mm

    rows, groups, n, k = sizes
    x, w, dy = _make(rows, groups, n, k, seed=rows)
    for kind in ("gaps", "router"):
        offsets = _offsets(rows, groups, kind, seed=n)
        owner = torch.bucketize(torch.arange(rows), offsets, right=True) - 1  # -1 or groups: none
        owner[owner == groups] = -1
        x.requires_grad_(True)
        y = grouped_mm(x, w, offsets.cuda())
        dx, = torch.autograd.grad(y, x, dy)
        x.requires_grad_(False)
        mine = w[owner.clamp_min(0).cuda()].to(F64) * (owner >= 0).cuda()[:, None, None]
        a, g = x.to(F64)[:, None], dy.to(F64)[:, None]
        _close(y, (a * mine).sum(2), (a * mine).abs().sum(2), k)
        _close(dx, (g.mT * mine).sum(1), (g.mT * mine).abs().sum(1), n)


@pytest.mark.parametrize("rows,groups,n,k", [(1, 1, 1, 1), (5, 3, 33, 7), (20, 8, 1288, 2051), (40, 8, 1287, 263),
                                             (100, 8, 520, 65), (9, 2, 40, 127), (300, 90, 264, 61)])
def test_few_rows_of_any_width(rows, groups, n, k):
    """Without gradients the weights and rows are read where they lie: NaN around them has no part."""
    from ops import _hip
    from ops.grouped_execution import grouped_mm

    assert _hip.query("ws_grouped_tile", rows, groups, n, k, NT) >= 5
    x, w, _ = _make(rows, groups, n, k, seed=k)
    offsets = _offsets(rows, groups, "router", seed=n)
    wide_x = torch.full((rows + 1, k + 3), float("nan"), dtype=BF16, device="cuda")
    wide_w = torch.full((groups, n + 1, k + 5), float("nan"), dtype=BF16, device="cuda")
    wide_x[:rows, 1:k + 1] = x
    wide_w[:, :n, 3:k + 3] = w
    with torch.no_grad():
        y = grouped_mm(wide_x[:rows, 1:k + 1], wide_w[:, :n, 3:k + 3], offsets.cuda())
        assert torch.equal(y, grouped_mm(x, w, offsets.cuda()))
        assert torch.equal(y, grouped_mm(x.T.contiguous().T, w.mT.contiguous().mT, offsets.cuda()))
    assert torch.equal(y, grouped_mm(x, w.requires_grad_(True), offsets.cuda()))  # (padded copies)
    _check(x, w.detach(), None, offsets, y.detach())


# Rows, groups, n, k of products that are cut in slices of the reduction, forward or to x.
SLICED = [(64, 2, 136, 2056), (100, 3, 72, 4000), (300, 2, 520, 3000), (513, 4, 264, 2304), (300, 3, 3000, 520),
          (200, 1, 1288, 5000), (300, 16, 520, 2056), (539, 1, 728, 11720), (1154, 1, 10248, 360), (2373, 1, 8640, 256),
          (100, 3, 4104, 2056), (90, 3, 2056, 136)]


def test_every_tile_is_cut():
    from ops import _hip

    found = set()
    for form in (NT, NN):
        for r, g, n, k in SLICED:
            sizes = (r, g, *((k, n) if form == NN else (n, k)), form)
            if _hip.query("ws_grouped_workspace_floats", *sizes):
                found.add((form, _hip.query("ws_grouped_tile", *sizes)))
    assert {(NT, 2), (NT, 3), (NT, 4), (NN, 2), (NN, 3), (NN, 4)} <= found, found


@pytest.mark.parametrize("kind", ["router", "gaps"])
@pytest.mark.parametrize("sizes", SLICED)
def test_slices(sizes, kind):
    from ops import _hip
    from ops.grouped_execution import grouped_mm

    rows, groups, n, k = sizes
    x, w, dy = _make(rows, groups, n, k, BF16, seed=rows + k)
    assert max(_hip.query("ws_grouped_workspace_floats", rows, groups, n, k, NT),
               _hip.query("ws_grouped_workspace_floats", rows, groups, k, n, NN)) > 0
    offsets = _offsets(rows, groups, kind, seed=n)
    x.requires_grad_(True)
    y = grouped_mm(x, w, offsets.cuda())
    dx, = torch.autograd.grad(y, x, dy)
    _check(x.detach(), w, dy, offsets, y, dx)
    again = grouped_mm(x, w, offsets.cuda())
    assert torch.equal(y, again) and torch.equal(dx, torch.autograd.grad(again, x, dy)[0])


def test_every_tile_is_reached():
    from ops import _hip

    found = {form: {_hip.query("ws_grouped_tile", r, g, *((k, n) if form == NN else (n, k)), form)
                    for r, g, n, k in SIZES} for form in (NT, NN, GRAD)}
    assert {0, 1, 2, 3, 4, 5, 6} <= found[NT], found
    assert {0, 1, 2, 3, 4} <= found[NN] and {0, 1, 3, 4} <= found[GRAD], found


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,groups,n,k", [(1, 1, 1, 1), (3, 2, 5, 7), (40, 3, 77, 130), (513, 4, 131, 67),
                                             (900, 3, 264, 100), (900, 3, 100, 264)])
def test_odd_widths(rows, groups, n, k, dtype):
    from ops.grouped_execution import grouped_mm

    x, w, dy = _make(rows, groups, n, k, dtype, seed=k)
    offsets = _offsets(rows, groups, "router", seed=k)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = grouped_mm(x, w, offsets.cuda())
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert y.is_contiguous() and dx.is_contiguous() and dw.is_contiguous()
    assert y.shape == dy.shape and dx.shape == x.shape and dw.shape == w.shape
    _check(x.detach(), w, dy, offsets, y, dx, dw)


@pytest.mark.parametrize("sizes", [(300, 2, 520, 3000), (512, 512, 264, 40), (40, 8, 1288, 263)])
def test_replays(sizes):
    """A captured product follows other rows and offsets, with eager work between the replays; slices,
    several tiles of a workgroup, rows read where they lie."""
    from ops.grouped_execution import grouped_mm

    rows, groups, n, k = sizes
    x, w, _ = _make(rows, groups, n, k)
    offsets = _offsets(rows, groups, "router").cuda()
    with torch.no_grad():
        grouped_mm(x, w, offsets)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = grouped_mm(x, w, offsets)
        for seed, kind in enumerate(("gaps", "one", "even", "router"), 1):
            x.copy_(_make(rows, groups, n, k, seed=seed)[0])
            offsets.copy_(_offsets(rows, groups, kind, seed))
            graph.replay()
            torch.cuda.synchronize()
            kept = y.clone()
            assert torch.equal(kept, grouped_mm(x, w, offsets)), kind


def test_layouts():
    """Row strides, odd offsets, transposed operands, an expanded gradient and expanded weights: the
    same bits as contiguous operands."""
    from ops.grouped_execution import grouped_mm

    rows, groups, n, k = 70, 3, 64, 72
    x, w, dy = _make(rows, groups, n, k)
    offsets = _offsets(rows, groups, "router").cuda()
    want = grouped_mm(x, w, offsets)
    wide = torch.full((rows, k + 16), float("nan"), dtype=BF16, device="cuda")
    for first in (0, 3, 8):
        wide[:, first:first + k] = x
        assert torch.equal(grouped_mm(wide[:, first:first + k], w, offsets), want)
    assert torch.equal(grouped_mm(x.t().contiguous().t(), w, offsets), want)
    assert torch.equal(grouped_mm(x, w.transpose(1, 2).contiguous().transpose(1, 2), offsets), want)
    many = torch.full((groups, n + 3, k + 8), float("nan"), dtype=BF16, device="cuda")
    many[:, :n, :k] = w
    assert torch.equal(grouped_mm(x, many[:, :n, :k], offsets), want)
    same = grouped_mm(x, w[:1].expand(groups, n, k), offsets)
    assert torch.equal(same, grouped_mm(x, w[:1].repeat(groups, 1, 1), offsets))
    strided = torch.stack([offsets, offsets], 1)[:, 1]
    assert torch.equal(grouped_mm(x, w, strided), want)
    leaf, leaf_w = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = torch.autograd.grad(grouped_mm(leaf, leaf_w, offsets).sum(), [leaf, leaf_w])
    again = torch.autograd.grad(grouped_mm(leaf, leaf_w, offsets), [leaf, leaf_w], torch.ones_like(dy))
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    shared = w[:1].clone().requires_grad_(True)  # a broadcast weight's gradient is the groups' sum
    one, = torch.autograd.grad(grouped_mm(x, shared.expand(groups, n, k), offsets), [shared], dy)
    g, a = dy.to(F64), x.to(F64)
    _close(one[0].float(), g.T @ a, g.abs().T @ a.abs(), rows + groups * 2 ** 16)


@pytest.mark.parametrize("want", ["x", "weight"])
def test_one_gradient(want):
    from ops.grouped_execution import grouped_mm

    x, w, dy = _make(130, 4, 136, 64, F32)
    offsets = _offsets(130, 4, "router").cuda()
    (x if want == "x" else w).requires_grad_(True)
    y = grouped_mm(x, w, offsets)
    got, = torch.autograd.grad(y, [x if want == "x" else w], dy)
    _check(x.detach(), w, dy, offsets.cpu(), y, **({"dx": got} if want == "x" else {"dw": got}))


def test_no_rows():
    from ops.grouped_execution import grouped_mm

    x, w, dy = _make(0, 3, 16, 24)
    w.requires_grad_(True)
    x.requires_grad_(True)
    y = grouped_mm(x, w, torch.zeros(4, dtype=torch.int64, device="cuda"))
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert y.shape == (0, 16) and dx.shape == (0, 24) and not dw.any()


@pytest.mark.parametrize("sizes", [(16, 6, 64, 256), (300, 6, 264, 256), (5000, 6, 512, 256), (150, 6, 264, 4096)])
def test_any_offsets_stay_inside(sizes):
    """Values that name rows that there are not, or name them twice, change no memory but the
    result's; rows behind y and beside it stay as they were."""
    from ops import _hip

    rows, groups, n, k = sizes
    x, w, dy = _make(rows, groups, n, k)
    wide = torch.full((rows + 2, n + 16), 7.0, dtype=BF16, device="cuda")
    dw = torch.full((groups + 1, n, k), 7.0, device="cuda")
    need = _hip.query_on(x, "ws_grouped_workspace_floats", rows, groups, n, k, NT)
    assert (need > 0) == (k == 4096)
    work = torch.full((need + 64,), 7.0, device="cuda")
    for values in ([0, 5, 3, rows, rows + 9, 2 ** 40, -4], [-2 ** 62] * 7, [2 ** 62] * 7,
                   [rows, 0, rows, 0, rows, 0, rows], [3] * 7):
        offsets = torch.tensor(values, device="cuda")
        _hip.call_on(x, "ws_grouped_mm", x.data_ptr(), k, w.data_ptr(), k, n * k, NT, offsets.data_ptr(),
                     groups, rows, n, k, wide[1:, 8:].data_ptr(), n + 16, work.data_ptr())
        _hip.call_on(x, "ws_grouped_weight_grad", dy.data_ptr(), n, x.data_ptr(), k, offsets.data_ptr(),
                     groups, rows, n, k, dw.data_ptr(), 1)
        assert (wide[0] == 7).all() and (wide[rows + 1] == 7).all()
        assert (wide[:, :8] == 7).all() and (wide[:, n + 8:] == 7).all() and (dw[groups] == 7).all()
        assert (work[need:] == 7).all()


def test_bad_values_stay_in_their_group():
    from ops.grouped_execution import grouped_mm

    rows, groups, n, k = 90, 3, 64, 128
    x, w, dy = _make(rows, groups, n, k)
    offsets = torch.tensor([0, 31, 31, 90], device="cuda")
    clean = grouped_mm(x, w, offsets)
    w[1] = float("nan")  # no rows
    x[40] = float("inf")
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = grouped_mm(x, w, offsets)
    rest = [t for t in range(rows) if t != 40]
    assert torch.equal(y[rest], clean[rest]) and not y[40].isfinite().all()
    _, dw = torch.autograd.grad(y, [x, w], dy)
    assert dw[0].isfinite().all() and not dw[1].any() and not dw[2].isfinite().all()


@pytest.mark.parametrize("odd", [False, True])
def test_python_form_gives_the_same_bits(odd, monkeypatch):
    from ops import _hip
    from ops.grouped_execution import grouped_mm

    n, k = (131, 77) if odd else (136, 72)
    x, w, dy = _make(200, 5, n, k, F32)
    offsets = _offsets(200, 5, "gaps").cuda()

    def run():
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = grouped_mm(a, b, offsets)
        return (y, *torch.autograd.grad(y, [a, b], dy))

    want = run()
    monkeypatch.setattr(_hip, "host_ops", lambda: None)
    for a, b in zip(run(), want):
        assert torch.equal(a, b)


def test_past_2_31_elements():
    """Rows, weights and gradients whose offsets pass 32 bits."""
    from ops.grouped_execution import grouped_mm

    rows, groups, n, k = 280000, 24, 11264, 8192
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn((rows, k), generator=g, device="cuda", dtype=BF16).requires_grad_(True)
    w = (0.02 * torch.randn((groups, n, k), generator=g, device="cuda", dtype=BF16)).requires_grad_(True)
    counts = torch.tensor([279000] + [0] * 21 + [400, 600])
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    y = grouped_mm(x, w, offsets.cuda())
    dy = torch.zeros((rows, n), dtype=BF16, device="cuda")
    dy[-600:] = torch.randn((600, n), generator=g, device="cuda", dtype=BF16)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    a, b, d = x.detach()[-600:].to(F64), w.detach()[-1].to(F64), dy[-600:].to(F64)
    _close(y[-600:], a @ b.T, a.abs() @ b.abs().T, k)
    _close(dx[-600:], d @ b, d.abs() @ b.abs(), n)
    _close(dw[-1], d.T @ a, d.abs().T @ a.abs(), 600)
    assert not dw[1:23].any() and not dx[:1000].any()
    a, b = x.detach()[278000:278100].to(F64), w.detach()[0].to(F64)
    _close(y[278000:278100], a @ b.T, a.abs() @ b.abs().T, k)
