"""Block quantization to e4m3 and the block-scaled product on the GPU, against 64-bit numpy."""
import numpy as np
import pytest
import torch

from fp8_reference import BLOCK, E8M0, F32, dequantize, quantize, values

pytestmark = pytest.mark.gpu
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
SCALES = [E8M0, F32]


def _fp8():
    from ops import fp8_execution

    return fp8_execution


def _matrix(rows, cols, dtype, seed, std=1.0):
    """Normal values with loud columns, an all-zero block, tiny and huge blocks."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * std
    x[:, ::37] *= 20.0
    x[: rows // 3, : cols // 4] = 0.0
    if cols > BLOCK:
        x[rows // 2:, BLOCK:2 * BLOCK] *= 1e-30
    if cols > 2 * BLOCK:
        x[rows // 2:, 2 * BLOCK:3 * BLOCK] *= 1e20
    return x.to(dtype).cuda()


def _same(got, want):
    np.testing.assert_array_equal(values(got), want)


SIZES = [(1, 1), (1, 128), (3, 129), (17, 7), (128, 128), (129, 300), (200, 513), (77, 1000)]


@pytest.mark.parametrize("scale_dtype", SCALES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantized_values_and_scales_are_exact(rows, cols, dtype, scale_dtype):
    """Scales and 8-bit values follow from the definition without any freedom: equal bits."""
    fp8 = _fp8()
    x = _matrix(rows, cols, dtype, rows * 1000 + cols)
    wide = values(x)
    q, scale, qt, scale_t = fp8.quantize_rows_and_columns(x, scale_dtype)
    want_q, want_scale = quantize(wide, scale_dtype)
    want_qt, want_scale_t = quantize(np.ascontiguousarray(wide.T), scale_dtype)
    for got, want in ((q, want_q), (scale, want_scale), (qt, want_qt), (scale_t, want_scale_t)):
        _same(got, want)
    for got, want in zip(fp8.quantize_rows(x, scale_dtype), (q, scale)):
        _same(got, values(want))
    for got, want in zip(fp8.quantize_columns(x, scale_dtype), (qt, scale_t)):
        _same(got, values(want))
    w, w_scale, wt, wt_scale = fp8.quantize_weight(x, scale_dtype)
    want_w, want_w_scale = quantize(wide, scale_dtype, BLOCK)
    for got, want in ((w, want_w), (w_scale, want_w_scale), (wt, want_w.T), (wt_scale, want_w_scale.T)):
        _same(got, want)


@pytest.mark.parametrize("scale_dtype", SCALES)
def test_quantization_of_views(scale_dtype):
    """Unaligned columns, odd row strides and transposed inputs give the same values."""
    fp8 = _fp8()
    base = _matrix(150, 411, BF16, 5)
    for view in (base[:, 3:300], base[1:, 8:200], base.T, base[::2]):
        want = fp8.quantize_rows_and_columns(view.contiguous(), scale_dtype)
        for got, expect in zip(fp8.quantize_rows_and_columns(view, scale_dtype), want):
            _same(got, values(expect))


@pytest.mark.parametrize("scale_dtype", SCALES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_bad_value_stays_in_its_block(bad, scale_dtype):
    fp8 = _fp8()
    x = _matrix(130, 300, BF16, 9, std=0.5)
    clean = [values(t) for t in fp8.quantize_rows(x, scale_dtype)]
    x[5, 140] = bad
    q, scale = (values(t) for t in fp8.quantize_rows(x, scale_dtype))
    assert np.isnan(dequantize(q, scale)[5, 140])
    if scale_dtype == E8M0:
        assert np.isnan(scale[5, 1])
    mask = np.ones_like(q, bool)
    mask[5, 128:256] = False
    np.testing.assert_array_equal(q[mask], clean[0][mask])


def _operands(m, n, k, scale_dtype, a_blocks, b_blocks, seed):
    fp8 = _fp8()
    x = _matrix(m, k, BF16, seed).clamp(-100, 100)
    w = torch.randn((n, k), generator=torch.Generator().manual_seed(seed + 1)).mul(0.05).cuda()
    a = fp8.quantize_weight(x, scale_dtype)[:2] if a_blocks else fp8.quantize_rows(x, scale_dtype)
    b = fp8.quantize_weight(w, scale_dtype)[:2] if b_blocks else fp8.quantize_rows(w, scale_dtype)
    return (*a, *b)


def _check(got, a, sa, b, sb):
    """Every output within its bound of the 64-bit product. The matrix instruction cuts each of
    the eight products of a group at 2^-13 of the largest one's power of two: at most
    8 * 2^-13 of the sum of magnitudes. FP32 sums: a product passes through at most
    16 additions in a block and one per block (2^-24 of the sum of magnitudes each, 2^-23 where
    the instruction truncates), and the FP32 scales' product is rounded once. Then one rounding
    to BF16 (half a step, 2^-8 relative)."""
    fa, fb = dequantize(values(a), values(sa)), dequantize(values(b), values(sb))
    want = fa @ fb.T
    size = np.abs(fa) @ np.abs(fb).T
    k = fa.shape[1]
    sums = (2.0 ** -10 + (k / BLOCK + 18) * 2.0 ** -23) * size
    bound = sums + (np.abs(want) + sums) * 2.0 ** -8 + 1e-38
    worst = np.max(np.abs(values(got) - want) / bound)
    assert worst <= 1.0, worst


PRODUCTS = [(1, 1, 1), (1, 5, 130), (3, 128, 128), (16, 64, 256), (17, 96, 640), (33, 200, 1000),
            (64, 260, 384), (129, 130, 131), (200, 512, 1024), (300, 257, 2048), (511, 264, 272),
            (520, 513, 400)]
KINDS = [(False, True), (False, False), (True, True)]


@pytest.mark.parametrize("scale_dtype", SCALES)
@pytest.mark.parametrize("a_blocks,b_blocks", KINDS)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k, a_blocks, b_blocks, scale_dtype):
    a, sa, b, sb = _operands(m, n, k, scale_dtype, a_blocks, b_blocks, m + n + k)
    _check(_fp8().fp8_mm(a, sa, b, sb), a, sa, b, sb)


@pytest.mark.parametrize("scale_dtype", SCALES)
@pytest.mark.parametrize("a_blocks,b_blocks", KINDS)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_exact_product(m, n, k, a_blocks, b_blocks, scale_dtype):
    """Integers of at most 2 in magnitude and power-of-two scales of one binade or two: every
    product and every sum (below 2^24 of the smallest unit) is exact, and so is the result up
    to its one rounding to BF16. A misplaced operand, k index or scale shows."""
    g = torch.Generator().manual_seed(m * n + k)
    kb = -(-k // BLOCK)

    def operand(rows, blocks):
        q = torch.randint(-2, 3, (rows, k), generator=g).float()
        r = -(-rows // BLOCK) if blocks else rows
        return q.to(E4M3).cuda(), torch.randint(-1, 2, (r, kb), generator=g).float().exp2()

    a, sa = operand(m, a_blocks)
    b, sb = operand(n, b_blocks)
    want = dequantize(values(a), values(sa)) @ dequantize(values(b), values(sb)).T
    want = torch.from_numpy(want).to(BF16)
    cast = (lambda s: (s.log2() + 127).to(torch.uint8).view(E8M0)) if scale_dtype == E8M0 else (lambda s: s)
    got = _fp8().fp8_mm(a, cast(sa).cuda(), b, cast(sb).cuda())
    assert torch.equal(got.cpu(), want)


# (m, n, k, tile of ws_fp8_mm_plan, split): every macro-tile, whole and in slices of the
# reduction, ragged in every dimension.
PLANNED = [(2937, 3001, 128, 0, False), (3300, 2700, 1000, 0, False), (3717, 4947, 688, 0, True),
           (1380, 3173, 128, 1, False), (198, 5393, 9232, 1, True), (1020, 3933, 2864, 2, False),
           (73, 5450, 9472, 2, True), (286, 6767, 128, 3, False), (285, 3444, 4368, 3, True),
           (34, 33, 160, 4, False), (37, 39, 1168, 4, True), (64, 2048, 5632, 4, True),
           (32, 37, 176, 5, False), (17, 2000, 2064, 5, False)]


@pytest.mark.parametrize("scale_dtype", SCALES)
@pytest.mark.parametrize("a_blocks,b_blocks", KINDS)
@pytest.mark.parametrize("m,n,k,tile,split", PLANNED)
def test_exact_product_on_every_tile(m, n, k, tile, split, a_blocks, b_blocks, scale_dtype):
    """As test_exact_product, the reference an FP32 product on the GPU: sums of at most 9472
    products of at most 16 in units of 1/4 need 21 bits, so FP32 holds them exactly."""
    import ctypes

    from ops import _hip

    splits = ctypes.c_int()
    plan = _hip.library().ws_fp8_mm_plan(m, n, -(-k // 16) * 16, BLOCK if b_blocks else 1,
                                         int(scale_dtype == F32), None, ctypes.byref(splits))
    if scale_dtype == F32 and not b_blocks and tile == 0:
        assert plan != 0  # no such kernel: the product runs on smaller tiles
    else:
        assert (plan, splits.value > 1) == (tile, split)
    g = torch.Generator("cuda").manual_seed(m + n + k)
    kb = -(-k // BLOCK)

    def operand(rows, blocks):
        q = torch.randint(-2, 3, (rows, k), generator=g, device="cuda").float()
        r = -(-rows // BLOCK) if blocks else rows
        scale = torch.randint(-1, 2, (r, kb), generator=g, device="cuda").float().exp2()
        wide = scale.repeat_interleave(BLOCK if blocks else 1, 0)[:rows]
        return q.to(E4M3), scale, q * wide.repeat_interleave(BLOCK, 1)[:, :k]

    a, sa, fa = operand(m, a_blocks)
    b, sb, fb = operand(n, b_blocks)
    cast = (lambda s: (s.log2() + 127).to(torch.uint8).view(E8M0)) if scale_dtype == E8M0 else (lambda s: s)
    guard = torch.full((m + 2, n), 3.0, dtype=BF16, device="cuda")
    got = _fp8().fp8_mm(a, cast(sa), b, cast(sb), out=guard[1:-1])
    assert torch.equal(got, (fa @ fb.T).to(BF16))
    assert bool((guard[0] == 3.0).all()) and bool((guard[-1] == 3.0).all())


@pytest.mark.parametrize("scale_dtype", SCALES)
def test_product_of_other_layouts(scale_dtype):
    """Operands by columns, odd strides and unaligned starts, scales in the other order, and an
    output inside a larger buffer, whose other elements stay."""
    fp8 = _fp8()
    a, sa, b, sb = _operands(130, 72, 272, scale_dtype, False, False, 4)
    want = fp8.fp8_mm(a, sa, b, sb)

    def byte_copy(t, view):
        raw = t.view(torch.uint8)
        out = view(raw.shape)
        out.copy_(raw)
        return out.view(t.dtype)

    columns = byte_copy(a, lambda s: torch.empty(s[::-1], dtype=torch.uint8, device="cuda").T)
    odd = byte_copy(b, lambda s: torch.empty((s[0], s[1] + 5), dtype=torch.uint8, device="cuda")[:, 3:3 + s[1]])
    if scale_dtype == E8M0:
        other_sa = byte_copy(sa, lambda s: torch.empty(s[::-1], dtype=torch.uint8, device="cuda").T)
        other_sb = byte_copy(sb, lambda s: torch.empty(s, dtype=torch.uint8, device="cuda"))
    else:
        other_sa, other_sb = sa.contiguous(), sb.contiguous()
    big = torch.full((140, 99), 7.0, dtype=BF16, device="cuda")
    got = fp8.fp8_mm(columns, other_sa, odd, other_sb, out=big[3:133, 5:77])
    assert torch.equal(got, want)
    big[3:133, 5:77] = 7.0
    assert bool((big == 7.0).all())


@pytest.mark.parametrize("m,n,k", [(3300, 2700, 1000), (3717, 4948, 688), (1380, 3172, 128), (1020, 3932, 2864),
                                   (286, 6764, 128), (285, 3444, 4368), (34, 36, 160), (17, 2004, 2064)])
def test_output_inside_a_wider_buffer(m, n, k):
    """Aligned columns of a larger matrix, half of a 16-byte piece at the end: every kernel leaves
    the columns beside them and the rows behind them as they were."""
    fp8 = _fp8()
    a, sa, b, sb = _operands(m, n, k, E8M0, False, True, m + n)
    want = fp8.fp8_mm(a, sa, b, sb)
    big = torch.full((m + 9, n + 24), 7.0, dtype=BF16, device="cuda")
    out = big[1:m + 1, 8:8 + n]
    assert fp8.fp8_mm(a, sa, b, sb, out=out).data_ptr() == out.data_ptr() and torch.equal(out, want)
    out.fill_(7.0)
    assert bool((big == 7.0).all())


def test_scaled_nan_reaches_its_row_only():
    fp8 = _fp8()
    x = _matrix(40, 256, BF16, 1, std=0.1)
    x[7, 200] = float("nan")
    w = torch.randn((48, 256), generator=torch.Generator().manual_seed(2)).cuda()
    b, sb = fp8.quantize_weight(w)[:2]
    out = fp8.fp8_mm(*fp8.quantize_rows(x), b, sb)
    assert bool(torch.isnan(out[7]).all())
    assert not bool(torch.isnan(torch.cat((out[:7], out[8:]))).any())


@pytest.mark.parametrize("scale_dtype", SCALES)
@pytest.mark.parametrize("weight_dtype", [F32, BF16])
@pytest.mark.parametrize("m,n,k", [(1, 24, 40), (130, 72, 200), (300, 264, 136)])
def test_linear_and_its_gradients(m, n, k, weight_dtype, scale_dtype):
    """The three products of a projection are the products of the operands' quantized values."""
    fp8 = _fp8()
    x = _matrix(m, k, BF16, 11).clamp(-50, 50).requires_grad_(True)
    w = (torch.randn((n, k), generator=torch.Generator().manual_seed(12)) * 0.1).to(weight_dtype)
    w = w.cuda().requires_grad_(True)
    dy = _matrix(m, n, BF16, 13).clamp(-50, 50)
    y = fp8.fp8_linear(x, w, scale_dtype)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert (y.dtype, dx.dtype, dw.dtype) == (BF16, BF16, weight_dtype)
    if weight_dtype == F32:  # FP32 sums of the BF16 tensors' products
        fdy, fx = values(dy), values(x)
        size = np.abs(fdy).T @ np.abs(fx)
        assert np.all(np.abs(values(dw) - fdy.T @ fx) <= (m + 2) * 2.0 ** -23 * size + 1e-38)
    else:
        _check(dw, *fp8.quantize_columns(dy, scale_dtype), *fp8.quantize_columns(x, scale_dtype))
    rows = fp8.quantize_rows
    w_q, w_s, wt_q, wt_s = fp8.quantize_weight(w, scale_dtype)
    _check(y, *rows(x, scale_dtype), w_q, w_s)
    _check(dx, *rows(dy, scale_dtype), wt_q, wt_s)
    only, = torch.autograd.grad(fp8.fp8_linear(x.detach(), w, scale_dtype), [w], dy)
    assert torch.equal(only, dw)
    only, = torch.autograd.grad(fp8.fp8_linear(x, w.detach(), scale_dtype), [x], dy)
    assert torch.equal(only, dx)
    folded = fp8.fp8_linear(x.detach().view(1, m, k), w, scale_dtype)
    assert folded.shape == (1, m, n) and torch.equal(folded[0], y)


@pytest.mark.parametrize("scale_dtype", SCALES)
def test_operands_past_two_gib(scale_dtype):
    """More than 2^31 elements: the last rows are quantized and multiplied as on their own."""
    fp8 = _fp8()
    rows, k = 2 ** 31 // 2048 + 5000, 2048
    x = torch.empty((rows, k), dtype=BF16, device="cuda").normal_()
    b, sb = fp8.quantize_weight(torch.randn((24, k), device="cuda"), scale_dtype)[:2]
    q, scale = fp8.quantize_rows(x, scale_dtype)
    tail = slice(rows - 5000, rows)
    own_q, own_scale = fp8.quantize_rows(x[tail], scale_dtype)
    assert torch.equal(q[tail].view(torch.uint8), own_q.view(torch.uint8))
    assert np.array_equal(values(scale[tail]), values(own_scale))
    got = fp8.fp8_mm(q, scale, b, sb)[tail]
    _check(got[-300:], own_q[-300:], own_scale[-300:], b, sb)
    qt, scale_t = fp8.quantize_columns(x.T, scale_dtype)  # rows of x.T: columns past 2^31
    assert torch.equal(qt[tail].view(torch.uint8), own_q.view(torch.uint8))


def test_products_in_a_captured_graph():
    """Quantization and both products replay with new inputs, and with eager work between."""
    fp8 = _fp8()
    x = _matrix(130, 384, BF16, 21).clamp(-9, 9)
    b, sb = fp8.quantize_weight(torch.randn((200, 384), device="cuda"))[:2]

    def step():
        return fp8.fp8_mm(*fp8.quantize_rows(x), b, sb)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        x.copy_(_matrix(130, 384, BF16, 30 + seed).clamp(-9, 9))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())


def test_product_inside_a_compiled_function():
    fp8 = _fp8()
    x = _matrix(130, 384, BF16, 21).clamp(-9, 9)
    b, sb = fp8.quantize_weight(torch.randn((200, 384), device="cuda"))[:2]

    def step(x):
        return fp8.fp8_mm(*fp8.quantize_rows(x * 2.0), b, sb) + 1.0

    assert torch.equal(torch.compile(step, backend="aot_eager")(x), step(x))


def test_python_launches_agree_with_the_native_ones(monkeypatch):
    from ops import _hip

    fp8 = _fp8()
    assert _hip.host_ops() is not None
    x, w = _matrix(130, 272, BF16, 3).clamp(-9, 9), _matrix(96, 272, F32, 4).clamp(-9, 9)

    def run():
        out = []
        for scale_dtype in SCALES:
            q = fp8.quantize_rows_and_columns(x, scale_dtype)
            b = fp8.quantize_weight(w, scale_dtype)
            out += [*q, *b, *fp8.quantize_columns(x, scale_dtype), fp8.fp8_mm(*q[:2], *b[:2])]
        return out

    native = run()
    monkeypatch.setattr(_hip, "host_ops", lambda: None)
    for a, b in zip(native, run()):
        assert a.dtype == b.dtype and a.shape == b.shape and np.array_equal(values(a), values(b))


def test_linear_saves_no_more_than_it_reads():
    """A BF16 weight's step keeps 8-bit copies only; a call without gradients keeps nothing;
    compiled calls give the eager values."""
    fp8 = _fp8()
    x, w = _matrix(64, 256, BF16, 1).clamp(-9, 9), torch.randn((128, 256), device="cuda").to(BF16)
    plain = fp8.fp8_linear(x, w)
    assert not plain.requires_grad
    x.requires_grad_(True)
    w.requires_grad_(True)
    kept = []

    def pack(t):
        kept.append(t)
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = fp8.fp8_linear(x, w)
    assert torch.equal(y, plain) and all(t.dtype == torch.uint8 for t in kept)
    dy = torch.randn_like(y)
    want = torch.autograd.grad(y, [x, w], dy)
    compiled = torch.compile(fp8.fp8_linear, fullgraph=True)
    out = compiled(x, w)
    assert torch.equal(out, plain)
    for a, b in zip(torch.autograd.grad(out, [x, w], dy), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("native", [True, False])
def test_refusals_on_the_gpu(native, monkeypatch):
    """The same errors from either host path, before any launch."""
    from ops import _hip

    fp8 = _fp8()
    if not native:
        monkeypatch.setattr(_hip, "host_ops", lambda: None)
    a, sa, b, sb = _operands(20, 40, 256, E8M0, False, True, 2)
    cases = [((a.view(torch.uint8), sa, b, sb), "float8_e4m3fn"), ((a, sa, b[:, :128], sb), "Expected a"),
             ((a, sa.view(torch.uint8), b, sb), "Scales are"), ((a, sa, b, values_f32(sb)), "float8_e8m0fnu"),
             ((a, sa[:, :1], b, sb), "one scale per row"), ((a, sa, b, sa), "one scale per row"),
             ((a, sa[:7], b, sb), "one scale per row"), ((a[:0], sa, b, sb), "non-empty"),
             ((a, sa.cpu(), b, sb), "scales on")]
    for args, match in cases:
        with pytest.raises(ValueError, match=match):
            fp8.fp8_mm(*args)
    for out in (torch.empty((20, 40), device="cuda"), torch.empty((20, 41), device="cuda", dtype=BF16),
                torch.empty((40, 20), device="cuda", dtype=BF16).T):
        with pytest.raises(ValueError, match="out must"):
            fp8.fp8_mm(a, sa, b, sb, out=out)
    for x, match in ((torch.zeros(4, 4, device="cuda", dtype=torch.float16), "BF16 or FP32"),
                     (torch.zeros(4, device="cuda"), "non-empty matrix"),
                     (torch.zeros((0, 4), device="cuda"), "non-empty matrix")):
        with pytest.raises(ValueError, match=match):
            fp8.quantize_rows(x)
    with pytest.raises(ValueError, match="Scales are"):
        fp8.quantize_rows(torch.zeros(4, 4, device="cuda"), torch.float16)


def values_f32(scale):
    return torch.from_numpy(values(scale)).float().cuda()
