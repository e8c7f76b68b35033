"""Residual addition with RMSNorm against the formulas in 64 bits (GPU).

Bounds count roundings: a result's own (half a step: eps / 2 of its type, relative), the FP32
arithmetic before it (2^-24 an operation), and FP32 sums of n terms (at most n 2^-24 of the terms'
magnitudes; a row's lanes add at most 32 terms each, then 8 levels of halving)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
EPS = 1e-5
U = 2.0 ** -24
LANE_TERMS = 32 + 8 + 4


def _make(rows, d, stream=BF16, seed=0, **kw):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, d), generator=g).to(BF16)
    residual = (3 * torch.randn((rows, d), generator=g)).to(stream)
    weight = 1 + 0.1 * torch.randn((d,), generator=g)
    dy = (1e-2 * torch.randn((rows, d), generator=g)).to(BF16)
    ds = (1e-2 * torch.randn((rows, d), generator=g)).to(stream)
    return [t.cuda() for t in (x, residual, weight, dy, ds)]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _formula(stream, weight, dy=None, ds=None):
    """(y, d, dweight, magnitudes of d's FP32 error, of dweight's) in 64 bits."""
    s, w = stream.to(F64), weight.to(F64)
    d = s.shape[1]
    r = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + EPS)
    y = s * r * w
    if dy is None:
        return y
    g = dy.to(F64) * w
    h = ds.to(F64) if ds is not None else torch.zeros_like(s)
    m = (g * s).mean(1, keepdim=True) * r * r
    grad = h + r * (g - s * m)
    # Each term carries rstd's error (a row sum's, halved by the root; three times in m) and a few
    # operations; m also the error of its own sum.
    own = h.abs() + r * g.abs() + (r * s * m).abs()
    along = r * s.abs() * r * r * (g * s).abs().mean(1, keepdim=True)
    z = dy.to(F64) * s * r
    return y, grad, z.sum(0), 3 * LANE_TERMS * U * own + LANE_TERMS * U * along, z.abs().sum(0)


def _close(got, want, bound):
    off = (got.to(F64) - want).abs()
    assert got.isfinite().all()
    assert (off <= bound).all(), (off / bound.clamp_min(1e-300)).max().item()


SHAPES = [(1, 1), (1, 2048), (3, 7), (5, 129), (64, 512), (33, 520), (1025, 1280), (1500, 1000),
          (2000, 2048), (7, 2056), (1100, 2049), (3, 4096), (1300, 5632), (2, 8191), (40, 8192)]


@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("rows,d", SHAPES)
def test_forward_and_backward(rows, d, stream):
    from ops.residual_norm import add_rmsnorm

    x, residual, weight, dy, ds = _make(rows, d, stream, seed=rows + d)
    leaves = [t.requires_grad_(True) for t in (x, residual, weight)]
    y, out = add_rmsnorm(x, residual, weight, EPS)
    assert out.dtype == stream and y.dtype == BF16
    assert torch.equal(out, (x.detach().float() + residual.detach().float()).to(stream))
    dx, dr, dw = torch.autograd.grad([y, out], leaves, [dy, ds])
    assert dx.dtype == BF16 and dr.dtype == stream and dw.dtype == F32
    want_y, want, want_w, near, near_w = _formula(out.detach(), weight.detach(), dy, ds)
    _close(y, want_y, want_y.abs() * (_half(BF16) + LANE_TERMS * U))
    _close(dx, want, want.abs() * _half(BF16) + near)
    _close(dr, want, want.abs() * _half(stream) + near)
    # A workgroup adds at most rows / 4 terms, the join at most 512 partial rows.
    _close(dw, want_w, near_w * U * (min(rows, -(-rows // 512) + 512) + LANE_TERMS))


@pytest.mark.parametrize("upstream", ["y", "stream"])
@pytest.mark.parametrize("stream", [BF16, F32])
def test_one_upstream_gradient(stream, upstream):
    from ops.residual_norm import add_rmsnorm

    x, residual, weight, dy, ds = _make(70, 640, stream, seed=3)
    leaves = [t.requires_grad_(True) for t in (x, residual, weight)]
    y, out = add_rmsnorm(x, residual, weight, EPS)
    if upstream == "stream":
        dx, dr, dw = torch.autograd.grad(out, leaves, ds, allow_unused=True)
        assert torch.equal(dx, ds.to(BF16)) and torch.equal(dr, ds) and dw is None
        return
    dx, dr, dw = torch.autograd.grad(y, leaves, dy)
    _, want, want_w, near, near_w = _formula(out.detach(), weight.detach(), dy)
    _close(dx, want, want.abs() * _half(BF16) + near)
    _close(dr, want, want.abs() * _half(stream) + near)
    _close(dw, want_w, near_w * U * (70 + LANE_TERMS))


def test_gradient_against_differences():
    """The FP32 stream's gradient against central differences of the formula in 64 bits."""
    from ops.residual_norm import add_rmsnorm

    x, residual, weight, dy, ds = _make(6, 48, F32, seed=5)
    residual.requires_grad_(True)
    weight.requires_grad_(True)
    y, out = add_rmsnorm(x, residual, weight, EPS)
    dr, dw = torch.autograd.grad([y, out], [residual, weight], [dy, ds])
    s0, w0 = out.detach().to(F64), weight.detach().to(F64)

    def loss(s, w):
        r = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + EPS)
        return (s * r * w * dy.to(F64)).sum() + (s * ds.to(F64)).sum()

    step = 1e-5
    for at in [(0, 0), (2, 17), (5, 47)]:
        e = torch.zeros_like(s0)
        e[at] = step
        slope = (loss(s0 + e, w0) - loss(s0 - e, w0)) / (2 * step)
        # Differences of values of about one lose 2^-53 / step; curvature adds step^2.
        assert abs(dr[at].item() - slope.item()) < 1e-8 + 1e-5 * abs(slope.item())
    for at in (0, 31):
        e = torch.zeros_like(w0)
        e[at] = step
        slope = (loss(s0, w0 + e) - loss(s0, w0 - e)) / (2 * step)
        assert abs(dw[at].item() - slope.item()) < 1e-8 + 1e-5 * abs(slope.item())


def _scales(scale):
    if scale.dtype == F32:
        return scale.to(F64)
    code = scale.view(torch.uint8).to(torch.int32)
    return torch.exp2(code.to(F64) - 127)


@pytest.mark.parametrize("scale_dtype", [E8M0, F32])
@pytest.mark.parametrize("stream", [BF16, F32, None])
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 2048), (2, 100), (70, 128), (1029, 1280), (1030, 1277),
                                    (9, 5632), (1025, 2064), (3, 8192)])
def test_quantized(rows, d, stream, scale_dtype):
    from ops.residual_norm import rmsnorm_quantize

    x, residual, weight, _, _ = _make(rows, d, stream or BF16, seed=rows * 7 + d)
    residual = residual if stream else None
    q, scale, out = rmsnorm_quantize(x, weight, EPS, residual=residual, scale_dtype=scale_dtype)
    blocks = -(-d // 128)
    assert q.shape == (rows, d) and q.dtype == E4M3
    assert scale.shape == (rows, blocks) and scale.dtype == scale_dtype
    want = x if residual is None else (x.float() + residual.float()).to(stream)
    assert torch.equal(out, want)
    y = _formula(out, weight)
    s = _scales(scale).repeat_interleave(128, 1)[:, :d]
    near = LANE_TERMS * U
    # e4m3: half a step relative, or half a subnormal step of 2^-9.
    _close(q.float().to(F64) * s, y, torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + near) + near * y.abs())
    padded = torch.zeros((rows, blocks * 128), dtype=F64, device="cuda")
    padded[:, :d] = y.abs()
    amax = padded.view(rows, blocks, 128).amax(2)
    got = _scales(scale)
    if scale_dtype == F32:
        assert ((got - amax / 448).abs() <= amax / 448 * (near + 4 * U)).all()
    else:
        assert (amax <= 448 * got * (1 + near)).all() and (amax * (1 + near) > 224 * got).all()


def test_quantized_rows_feed_the_product():
    """Padded views as fp8_mm takes them, at a width that is no multiple of 16."""
    from ops.fp8_execution import fp8_mm, quantize_rows, quantize_weight
    from ops.residual_norm import rmsnorm_quantize

    x, residual, weight, _, _ = _make(20, 200, seed=1)
    w = torch.randn((64, 200), generator=torch.Generator().manual_seed(2)).cuda() * 0.1
    b, b_scale, _, _ = quantize_weight(w)
    q, scale, out = rmsnorm_quantize(x, weight, EPS, residual=residual)
    assert torch.equal(fp8_mm(q, scale, b, b_scale), fp8_mm(q.clone(), scale.clone(), b, b_scale))
    want_q, want_scale = quantize_rows(_formula(out, weight).float())
    assert (scale.view(torch.uint8) == want_scale.view(torch.uint8)).float().mean() > 0.99
    assert (q.view(torch.uint8) == want_q.view(torch.uint8)).float().mean() > 0.99


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_bad_values_stay_in_their_row(bad):
    from ops.residual_norm import add_rmsnorm, rmsnorm_quantize

    x, residual, weight, _, _ = _make(6, 300, seed=4)
    x[2, 5] = bad
    y, out = add_rmsnorm(x, residual, weight, EPS)
    rest = [0, 1, 3, 4, 5]
    assert y[rest].isfinite().all() and not y[2].isfinite().all()
    q, scale, _ = rmsnorm_quantize(x, weight, EPS, residual=residual)
    assert q[rest].float().isfinite().all() and (scale[rest].view(torch.uint8) < 255).all()
    assert scale[2, 0].view(torch.uint8) == 255


def test_zero_rows_are_zeros():
    from ops.residual_norm import add_rmsnorm, rmsnorm_quantize

    x = torch.zeros((3, 256), dtype=BF16, device="cuda")
    weight = torch.ones(256, device="cuda")
    y, out = add_rmsnorm(x, x, weight, EPS)
    assert not y.any() and not out.any()
    q, scale, _ = rmsnorm_quantize(x, weight, EPS, residual=x)
    assert not q.float().any()
    y, out = add_rmsnorm(x[:0], x[:0], weight, EPS)
    assert y.shape == out.shape == (0, 256)
    leaf = x[:0].clone().requires_grad_(True)
    w = weight.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(add_rmsnorm(leaf, x[:0], w)[0].sum(), [leaf, w])
    assert dx.shape == (0, 256) and not dw.any()


@pytest.mark.parametrize("stream", [BF16, F32])
def test_layouts(stream):
    """Leading dimensions, row strides, odd offsets, a transposed operand, an expanded gradient:
    the same bits as contiguous operands."""
    from ops.residual_norm import add_rmsnorm, rmsnorm_quantize

    x, residual, weight, dy, ds = _make(24, 320, stream, seed=8)
    want = add_rmsnorm(x, residual, weight, EPS)
    want_q = rmsnorm_quantize(x, weight, EPS, residual=residual)

    def layouts(t):
        wide = torch.full((24, 333), float("nan"), dtype=t.dtype, device="cuda")
        for first in (0, 1, 8):
            wide[:, first:first + 320] = t
            yield wide[:, first:first + 320].clone(memory_format=torch.preserve_format) if first == 8 else wide[:, first:first + 320]
        yield t.t().contiguous().t()
        yield t.view(2, 3, 4, 320)

    for a in layouts(x):
        for r in layouts(residual):
            r, shaped = r.reshape(a.shape), a.shape
            y, out = add_rmsnorm(a, r, weight, EPS)
            assert y.shape == shaped and y.is_contiguous() and out.is_contiguous()
            assert torch.equal(y.view(24, 320), want[0]) and torch.equal(out.view(24, 320), want[1])
            q, scale, out = rmsnorm_quantize(a, weight, EPS, residual=r)
            assert torch.equal(q.view(torch.uint8), want_q[0].view(torch.uint8))
            assert torch.equal(scale.view(torch.uint8), want_q[1].view(torch.uint8))
    leaf = x.clone().requires_grad_(True)
    got, = torch.autograd.grad(add_rmsnorm(leaf, residual, weight, EPS)[0].sum(), [leaf])
    again, = torch.autograd.grad(add_rmsnorm(leaf, residual, weight, EPS)[0], [leaf], torch.ones_like(x))
    assert torch.equal(got, again)


def test_weight_types():
    from ops.residual_norm import add_rmsnorm

    x, residual, weight, dy, _ = _make(24, 320, seed=9)
    w = weight.to(BF16).requires_grad_(True)
    y, _ = add_rmsnorm(x, residual, w, EPS)
    wide = w.detach().float().requires_grad_(True)
    want, _ = add_rmsnorm(x, residual, wide, EPS)
    assert torch.equal(y, want)
    got, = torch.autograd.grad(y, [w], dy)
    full, = torch.autograd.grad(want, [wide], dy)
    assert got.dtype == BF16 and torch.equal(got, full.to(BF16))
    strided = torch.stack([weight, weight], 1)[:, 0]
    assert torch.equal(add_rmsnorm(x, residual, strided, EPS)[0], add_rmsnorm(x, residual, weight, EPS)[0])


@pytest.mark.parametrize("stream", [BF16, F32])
def test_python_form_gives_the_same_bits(stream, monkeypatch):
    from ops import _hip
    from ops.residual_norm import add_rmsnorm, rmsnorm_quantize

    def run():
        x, residual, weight, dy, ds = _make(130, 1280, stream, seed=10)
        leaves = [t.requires_grad_(True) for t in (x, residual, weight)]
        y, out = add_rmsnorm(x, residual, weight, EPS)
        grads = torch.autograd.grad([y, out], leaves, [dy, ds])
        quantized = rmsnorm_quantize(x, weight, EPS, residual=residual, scale_dtype=F32)
        plain = rmsnorm_quantize(x, weight, EPS)
        return [y, out, *grads, *(t.view(torch.uint8) if t.dtype in (E4M3, E8M0) else t
                                  for t in (*quantized, *plain))]

    want = run()
    monkeypatch.setattr(_hip, "host_ops", lambda: None)
    for a, b in zip(run(), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("scale_dtype", [E8M0, F32])
def test_more_rows_than_one_launch_takes(scale_dtype):
    from ops.residual_norm import add_rmsnorm, rmsnorm_quantize

    rows, d = 4 * 2 ** 20 + 5, 8
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn((rows, d), generator=g, device="cuda").to(BF16)
    residual = torch.randn((rows, d), generator=g, device="cuda")
    weight = torch.randn(d, generator=g, device="cuda")
    y, out = add_rmsnorm(x, residual, weight, EPS)
    assert torch.equal(out, x.float() + residual)
    want = _formula(out, weight)
    _close(y, want, want.abs() * (_half(BF16) + LANE_TERMS * U))
    q, scale, out = rmsnorm_quantize(x, weight, EPS, residual=residual, scale_dtype=scale_dtype)
    s = _scales(scale).expand(rows, d)
    near = LANE_TERMS * U
    _close(q.float().to(F64) * s, want, torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + near) + near * want.abs())


def test_past_2_31_elements():
    from ops.residual_norm import add_rmsnorm

    rows, d = 1050000, 2048
    x = torch.randn((rows, d), dtype=BF16, device="cuda")
    residual = torch.randn((rows, d), dtype=BF16, device="cuda")
    weight = torch.randn(d, device="cuda").requires_grad_(True)
    x.requires_grad_(True)
    y, out = add_rmsnorm(x, residual, weight, EPS)
    dx, dw = torch.autograd.grad(y, [x, weight], residual)
    for part in (slice(0, 4), slice(rows // 2, rows // 2 + 4), slice(rows - 4, rows)):
        leaf = x.detach()[part].clone().requires_grad_(True)
        small, stream = add_rmsnorm(leaf, residual[part], weight, EPS)
        assert torch.equal(out[part], stream)
        _close(y[part], _formula(stream.detach(), weight.detach()),
               _formula(stream.detach(), weight.detach()).abs() * (_half(BF16) + LANE_TERMS * U))
        _, want, _, near, _ = _formula(stream.detach(), weight.detach(), residual[part])
        _close(dx[part], want, want.abs() * _half(BF16) + near)
    assert dw.isfinite().all()
