"""Token scores on the GPU against 64-bit arithmetic on the CPU."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
IGNORED = -100
U = 2.0 ** -24


def _scores():
    from ops import token_scores

    return token_scores


def _reference(logits, tokens, temperature, g=None, h=None):
    """(logprob, entropy, logp, dlogits) of 64-bit logits on the CPU."""
    scaled = logits.to(F64).cpu() / temperature
    tokens = tokens.cpu()
    logp = torch.log_softmax(scaled, -1)
    p = logp.exp()
    safe = torch.where(p > 0, logp, torch.zeros_like(logp))
    entropy = -(p * safe).sum(-1)
    valid = tokens != IGNORED
    index = tokens.clamp_min(0)[:, None]
    logprob = torch.where(valid, logp.gather(1, index)[:, 0], torch.zeros_like(entropy))
    if g is None:
        return logprob, entropy, logp, None
    g, h = g.to(F64).cpu() * valid, h.to(F64).cpu()
    grad = torch.zeros_like(p).scatter_(1, index, g[:, None]) - p * g[:, None]
    grad -= h[:, None] * p * (safe + entropy[:, None])
    return logprob, entropy, logp, grad / temperature


def _bounds(logits, temperature, extra=0.0):
    """(lse and log probability, entropy) error bounds. R bounds the finite scaled logits'
    magnitudes; `extra` is the logits' own error. Each e^x, |x| <= 2 R, has a relative error of
    at most (3 R + 2) 2^-23 (x and x log2 e rounded, the hardware's exponential); a sum passes
    at most 64 additions; the logarithm, the final difference and the rescalings of parts add
    a few roundings of lse's size."""
    finite = logits[torch.isfinite(logits)].double()
    r = float(finite.abs().max()) / temperature if finite.numel() else 0.0
    r += np.log(logits.shape[1])
    rel = (3 * r + 2) * 2 * U + 64 * U + extra
    score = rel + 8 * r * U + extra
    return score, (1 + 2 * r) * 2 * rel + 8 * r * U, rel


def _logits(rows, vocab, dtype, seed, std=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g) * std).to(dtype)


def _tokens(rows, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    if rows > 2:
        tokens[1] = IGNORED
    return tokens


def _top(logits, k):
    """Ids of the k largest logits, equal ones by the lowest id."""
    x = logits.float().numpy().astype(np.float64)
    return np.stack([np.lexsort((np.arange(x.shape[1]), -row))[:k] for row in x])


def _near(got, want, tol):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    same = torch.isnan(got) == torch.isnan(want)
    assert bool(same.all())
    ok = ~torch.isnan(want)
    worst = float((got - want)[ok].abs().max()) if bool(ok.any()) else 0.0
    assert worst <= tol, (worst, tol)


SIZES = [(1, 1), (2, 3), (3, 64), (1, 2048), (5, 2049), (2, 8192), (3, 8193), (700, 300),
         (600, 9001), (1, 40000), (2, 140001), (1, 524288)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_scores_and_likeliest_tokens(rows, vocab, temperature, dtype):
    ts = _scores()
    logits, tokens = _logits(rows, vocab, dtype, rows + vocab), _tokens(rows, vocab, vocab)
    logprob, entropy, logp, _ = _reference(logits, tokens, temperature)
    score_tol, entropy_tol, _rel = _bounds(logits, temperature)
    for k in sorted({0, 1, min(8, vocab), min(64, vocab)}):
        got = ts.token_scores(logits.cuda(), tokens.cuda(), k, temperature)
        _near(got.logprob, logprob, score_tol)
        _near(got.entropy, entropy, entropy_tol)
        ids = _top(logits, k)
        np.testing.assert_array_equal(got.top_ids.cpu().numpy(), ids)
        _near(got.top_logprobs, logp.gather(1, torch.from_numpy(ids)), score_tol)


def _special(name, rows, vocab):
    """Rows whose largest logits are hard to tell or to find."""
    x = _logits(rows, vocab, F32, 7)
    if name == "ties":
        x = (x * 2).round() / 2
    elif name == "equal":
        x = torch.full_like(x, 1.5)
    elif name == "zeros":  # -0 and 0 are one value
        x = torch.where(x > 0, 0.0, -0.0)
    elif name == "ascending":
        x = torch.arange(vocab).float().mul(1e-3).expand(rows, vocab).contiguous()
    elif name == "crowded":  # one group of threads low: nearly every other logit is a candidate
        x = x.abs()
        x[:, (torch.arange(vocab) % 2048) < 32] = -5.0
    elif name == "masked":
        x[:, torch.arange(vocab) % 97 != 5] = -float("inf")
    elif name == "one":
        x.fill_(-float("inf"))
        x[:, vocab // 2] = 2.0
    return x


@pytest.mark.parametrize("rows,vocab", [(3, 5000), (300, 16500), (1, 70000)])
@pytest.mark.parametrize("name", ["ties", "equal", "zeros", "ascending", "crowded", "masked", "one"])
def test_likeliest_tokens_of_special_rows(name, rows, vocab):
    ts = _scores()
    logits = _special(name, rows, vocab)
    tokens = torch.full((rows,), vocab // 2)
    logprob, entropy, logp, _ = _reference(logits, tokens, 1.0)
    score_tol, entropy_tol, _rel = _bounds(logits, 1.0)
    for dtype in (F32, BF16):
        if dtype == BF16 and name in ("crowded", "ascending"):
            continue  # these values are not BF16's
        x = logits.to(dtype)
        if dtype == BF16:
            logprob, entropy, logp, _ = _reference(x, tokens, 1.0)
        for k in (1, 20, 64):
            got = ts.token_scores(x.cuda(), tokens.cuda(), k)
            ids = _top(x, k)
            np.testing.assert_array_equal(got.top_ids.cpu().numpy(), ids)
            want = logp.gather(1, torch.from_numpy(ids))
            finite = torch.isfinite(want)
            top = got.top_logprobs.cpu().double()
            assert torch.equal(torch.isfinite(top), finite)
            _near(torch.where(finite, top, 0.0), torch.where(finite, want, 0.0), score_tol)
            inf = ~torch.isfinite(logprob)
            _near(got.logprob.cpu().masked_fill(inf, 0.0), logprob.masked_fill(inf, 0.0), score_tol)
            assert torch.equal(torch.isinf(got.logprob.cpu()), inf)
            _near(got.entropy, entropy, entropy_tol)


def test_rows_without_a_score():
    """All -inf: NaN, ids still valid. Tokens outside the vocabulary: NaN. Neighbours keep theirs."""
    ts = _scores()
    logits = _logits(6, 5000, F32, 3)
    clean = ts.token_scores(logits.cuda(), torch.arange(6).cuda(), 4)
    logits[2] = -float("inf")
    tokens = torch.tensor([0, 5000, 2, -1, IGNORED, 5])
    x = logits.cuda().requires_grad_(True)
    got = ts.token_scores(x, tokens.cuda(), 4)
    assert torch.isnan(got.logprob).tolist() == [False, True, True, True, False, False]
    assert torch.isnan(got.entropy).tolist() == [False, False, True, False, False, False]
    assert got.top_ids[2].tolist() == [0, 1, 2, 3] and float(got.logprob[4].detach()) == 0.0
    for i in (0, 5):
        assert torch.equal(got.logprob[i], clean.logprob[i])
        assert torch.equal(got.top_ids[i], clean.top_ids[i])
    up = torch.tensor([0.5, 0.0, 0.0, 0.0, 3.0, -1.0]).cuda()
    dx, = torch.autograd.grad(got.logprob, [x], up)
    assert not bool(torch.isnan(dx[[0, 2, 4, 5]]).any())
    assert not bool(dx[2].any()) and not bool(dx[4].any())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(1, 5), (3, 2047), (40, 3001), (130, 8200)])
def test_gradient_of_the_logits(rows, vocab, dtype):
    ts = _scores()
    logits, tokens = _logits(rows, vocab, dtype, 5, std=2.0), _tokens(rows, vocab, 6)
    logits[:, ::7] = -float("inf")
    keep = tokens.clamp_min(0)
    logits[torch.arange(rows), keep] = 1.0
    gen = torch.Generator().manual_seed(8)
    g, h = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen)
    for temperature in (1.0, 1.3):
        _, entropy, logp, want = _reference(logits, tokens, temperature, g, h)
        score_tol, entropy_tol, rel = _bounds(logits, temperature)
        x = logits.cuda().requires_grad_(True)
        got = ts.token_scores(x, tokens.cuda(), 0, temperature)
        dx, = torch.autograd.grad([got.logprob, got.entropy], [x], [g.cuda(), h.cuda()])
        assert dx.dtype == dtype
        p = logp.exp()
        surprise = torch.where(p > 0, logp.abs(), torch.zeros_like(p)) + entropy[:, None]
        size = p * (g.abs()[:, None] + h.abs()[:, None] * surprise) / temperature
        bound = size * (rel + score_tol + 16 * U) + p * h.abs()[:, None] * (score_tol + entropy_tol) / temperature
        bound = bound + (torch.finfo(dtype).eps / 2 + 4 * U) * (want.abs() + bound) + 1e-30
        worst = float(((dx.double().cpu() - want).abs() / bound).max())
        assert worst <= 1.0, worst


def test_gradient_against_differences():
    """Central differences of the 64-bit scores along random directions, step 1e-4: the
    third-order term is below 1e-6 of a score's scale."""
    ts = _scores()
    logits, tokens = _logits(6, 50, F32, 2, std=1.0), _tokens(6, 50, 3)
    g, h = torch.linspace(-1, 1, 6), torch.linspace(0.5, -0.7, 6)
    x = logits.cuda().requires_grad_(True)
    got = ts.token_scores(x, tokens.cuda())
    dx, = torch.autograd.grad([got.logprob, got.entropy], [x], [g.cuda(), h.cuda()])

    def total(values):
        logprob, entropy, _, _ = _reference(values, tokens, 1.0)
        return float((logprob * g + entropy * h).sum())

    for seed in range(4):
        v = torch.randn(6, 50, generator=torch.Generator().manual_seed(seed)).double()
        want = (total(logits.double() + 1e-4 * v) - total(logits.double() - 1e-4 * v)) / 2e-4
        assert abs(float((dx.double().cpu() * v).sum()) - want) <= 2e-5


def test_one_of_the_two_gradients_and_broadcast_upstream():
    ts = _scores()
    logits, tokens = _logits(9, 700, F32, 4).cuda(), _tokens(9, 700, 4).cuda()
    x = logits.clone().requires_grad_(True)
    one, = torch.autograd.grad(ts.token_scores(x, tokens).logprob.sum(), [x])
    ones, zeros = torch.ones(9).cuda(), torch.zeros(9).cuda()
    got = ts.token_scores(x, tokens)
    both, = torch.autograd.grad([got.logprob, got.entropy], [x], [ones, zeros])
    assert torch.equal(one, both)
    only, = torch.autograd.grad(ts.token_scores(x, tokens).entropy.sum(), [x])
    got = ts.token_scores(x, tokens)
    both, = torch.autograd.grad([got.logprob, got.entropy], [x], [zeros, ones])
    assert torch.equal(only, both)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logits_of_other_strides(dtype):
    ts = _scores()
    base = _logits(40, 3007, dtype, 1).cuda()
    for view in (base[:, 5:2900], base[::3, 1:], base.T[:30], base[:7].expand(7, 3007)):
        tokens = torch.arange(view.shape[0]).cuda() % view.shape[1]
        k = min(5, view.shape[1])
        want = ts.token_scores(view.contiguous(), tokens, k)
        for a, b in zip(ts.token_scores(view, tokens, k), want):
            assert torch.equal(a, b)


def test_empty_batch():
    ts = _scores()
    x = torch.empty((0, 100), device="cuda", requires_grad=True)
    got = ts.token_scores(x, torch.empty(0, dtype=torch.int64, device="cuda"), 3)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 3)
    dx, = torch.autograd.grad(got.logprob.sum(), [x])
    assert dx.shape == (0, 100)
    w = torch.randn(64, 16, device="cuda").to(BF16).requires_grad_(True)
    hidden = torch.empty((0, 16), device="cuda", dtype=BF16, requires_grad=True)
    logprob, _ = ts.linear_token_scores(hidden, w, torch.empty(0, dtype=torch.int64, device="cuda"))
    dh, dw = torch.autograd.grad(logprob.sum(), [hidden, w])
    assert dh.shape == (0, 16) and not bool(dw.any())


HEADS = [(1, 8, 5), (3, 64, 130), (2100, 64, 2056), (700, 72, 1501), (130, 40, 517), (257, 136, 1000), (300, 100, 264), (70, 256, 2304)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,d,vocab", HEADS)
def test_head_scores_and_gradients(rows, d, vocab, dtype):
    ts = _scores()
    gen = torch.Generator().manual_seed(rows + vocab)
    hidden = torch.randn((rows, d), generator=gen).to(BF16)
    weight = (torch.randn((vocab, d), generator=gen) * (2.0 / d ** 0.5)).to(BF16)
    tokens = _tokens(rows, vocab, 2)
    g, h = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen) * 0.3
    fh, fw = hidden.double(), weight.double()
    logits = fh @ fw.T
    # FP32 sums of d exact products, in any order.
    extra = (d + 2) * U * float((fh.abs() @ fw.abs().T).max())
    for temperature, chunk in ((1.0, 8192), (0.8, 96)):
        logprob, entropy, logp, grad = _reference(logits, tokens, temperature, g, h)
        score_tol, entropy_tol, rel = _bounds(logits, temperature, 2 * extra / temperature)
        a = hidden.to(dtype).cuda().requires_grad_(True)
        w = weight.to(dtype).cuda().requires_grad_(True)
        got = ts.linear_token_scores(a, w, tokens.cuda(), temperature, chunk)
        _near(got[0], logprob, score_tol)
        _near(got[1], entropy, entropy_tol)
        dh, dw = torch.autograd.grad(got, [a, w], [g.cuda(), h.cuda()])
        assert (dh.dtype, dw.dtype) == (dtype, dtype)
        p = logp.exp()
        size = p * (g.abs()[:, None] + h.abs()[:, None] * (logp.abs() + entropy[:, None])) / temperature
        err = size * (rel + score_tol + 16 * U) + p * h.abs()[:, None] * (score_tol + entropy_tol) / temperature
        # The BF16 rounding of the logit gradients (half a step, 2^-8 of a value at most), FP32
        # sums, and the rounding of the result (dHidden is BF16 whatever the operand's type).
        err = err + (grad.abs() + err) * 2.0 ** -8
        for out, want, bound, terms, final in (
                (dh, grad @ fw, err @ fw.abs(), grad.abs() @ fw.abs() * (vocab + 2), 2.0 ** -8),
                (dw, grad.T @ fh, err.T @ fh.abs(), grad.abs().T @ fh.abs() * (rows + 2),
                 torch.finfo(dtype).eps / 2)):
            bound = bound + terms * U
            bound = bound + (want.abs() + bound) * final + 1e-30
            worst = float(((out.double().cpu() - want).abs() / bound).max())
            assert worst <= 1.0, worst
        only, = torch.autograd.grad(ts.linear_token_scores(a.detach(), w, tokens.cuda(), temperature,
                                                           chunk), [w], [g.cuda(), h.cuda()])
        assert torch.equal(only, dw)


def test_head_operands_of_other_strides_and_bad_tokens():
    ts = _scores()
    hidden = torch.randn((33, 90), device="cuda").to(BF16)[:, 3:75]
    weight = torch.randn((72, 300), device="cuda").to(BF16).T
    tokens = torch.arange(33, device="cuda")
    tokens[4], tokens[5], tokens[6] = 300, -7, IGNORED
    want = ts.linear_token_scores(hidden.contiguous(), weight.contiguous(), tokens)
    got = ts.linear_token_scores(hidden, weight, tokens)
    for a, b in zip(got, want):
        assert torch.equal(torch.nan_to_num(a, 7.0), torch.nan_to_num(b, 7.0))
    assert torch.isnan(got[0]).nonzero()[:, 0].tolist() == [4, 5] and float(got[0][6]) == 0.0
    assert not bool(torch.isnan(got[1]).any())


def test_head_of_a_large_vocabulary():
    """More than 2^31 logits in five default chunks: scores and gradients of every row, against
    64 bits 200 rows at a time. `extra`: the logits' own error, FP32 sums of d products, and 64
    more additions per sum than _bounds counts. A gradient's FP32 sum of n terms is off by at
    most n U of the terms' magnitudes."""
    ts = _scores()
    rows, d, vocab = 4100, 8, 524288
    gen = torch.Generator().manual_seed(3)
    hidden = torch.randn((rows, d), generator=gen).to(BF16).cuda().requires_grad_(True)
    weight = torch.randn((vocab, d), generator=gen).to(BF16).cuda().requires_grad_(True)
    tokens = torch.randint(0, vocab, (rows,), generator=gen).cuda()
    tokens[5] = IGNORED
    up_g, up_h = torch.randn(rows, generator=gen).cuda(), torch.randn(rows, generator=gen).cuda()
    logprob, entropy = ts.linear_token_scores(hidden, weight, tokens)
    dh, dw = torch.autograd.grad([logprob, entropy], [hidden, weight], [up_g, up_h])
    logprob, entropy = logprob.detach(), entropy.detach()
    wide, want_dw, dw_tol = weight.detach().double(), 0.0, 0.0
    for a in range(0, rows, 200):
        part = slice(a, a + 200)
        x = hidden.detach()[part].double()
        logits = x @ wide.T
        extra = 2 * (d + 2) * U * float((x.abs() @ wide.abs().T).max()) + 64 * U
        score_tol, entropy_tol, rel = _bounds(logits, 1.0, extra)
        logp = torch.log_softmax(logits, -1)
        p, valid, index = logp.exp(), tokens[part] != IGNORED, tokens[part].clamp_min(0)[:, None]
        want_e = -(p * logp).sum(-1)
        assert float((logprob[part] - logp.gather(1, index)[:, 0] * valid).abs().max()) <= score_tol
        assert float((entropy[part] - want_e).abs().max()) <= entropy_tol
        g, h = (up_g[part].double() * valid)[:, None], up_h[part].double()[:, None]
        dl = -p * (g + h * (logp + want_e[:, None]))
        dl.scatter_add_(1, index, g)
        err = p * (g.abs() + h.abs() * (logp.abs() + want_e[:, None])) * (rel + score_tol + 16 * U)
        err += p * h.abs() * (score_tol + entropy_tol)
        err += (dl.abs() + err) * 2.0 ** -8
        err.scatter_add_(1, index, g.abs() * (4 * U + 2.0 ** -8))
        want = dl @ wide
        tol = err @ wide.abs() + vocab * U * ((dl.abs() + err) @ wide.abs())
        assert bool(((dh[part].double() - want).abs() <= tol + (want.abs() + tol) * 2.0 ** -8).all())
        want_dw = want_dw + dl.T @ x
        dw_tol = dw_tol + err.T @ x.abs() + rows * U * ((dl.abs() + err).T @ x.abs())
    tol = dw_tol + (want_dw.abs() + dw_tol) * 2.0 ** -8 + 1e-30
    assert bool(((dw.double() - want_dw).abs() <= tol).all())


def test_logits_past_two_gib():
    """More than 2^31 logits: the last rows are scored, and their gradient written, as on their
    own."""
    ts = _scores()
    rows, vocab = 4100, 524288
    x = torch.empty((rows, vocab), dtype=BF16, device="cuda").normal_().requires_grad_(True)
    tokens = torch.arange(rows, device="cuda") * 127
    g, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    got = ts.token_scores(x, tokens, 5)
    dx, = torch.autograd.grad([got.logprob, got.entropy], [x], [g, h])
    tail = slice(rows - 600, rows)  # as many rows as take the same parts
    own = x.detach()[tail].clone().requires_grad_(True)
    alone = ts.token_scores(own, tokens[tail], 5)
    want, = torch.autograd.grad([alone.logprob, alone.entropy], [own], [g[tail], h[tail]])
    for a, b in zip(got, alone):
        assert torch.equal(a[tail], b)
    assert torch.equal(dx[tail], want)


def test_scores_in_a_captured_graph():
    """Forward and backward from logits, and the head's forward, replayed with new inputs and
    eager work between the replays."""
    ts = _scores()
    logits = _logits(5, 20000, BF16, 1).cuda()
    tokens = _tokens(5, 20000, 1).cuda()
    hidden = torch.randn((40, 64), device="cuda").to(BF16)
    weight = torch.randn((500, 64), device="cuda").to(BF16)
    head_tokens = torch.arange(40, device="cuda")
    up = torch.randn(5, device="cuda")

    def step():
        x = logits.detach().requires_grad_(True)
        got = ts.token_scores(x, tokens, 8)
        dx, = torch.autograd.grad([got.logprob, got.entropy], [x], [up, up])
        return (*got, dx, *ts.linear_token_scores(hidden, weight, head_tokens))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        logits.copy_(_logits(5, 20000, BF16, 40 + seed))
        hidden.copy_(torch.randn((40, 64), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_scores_inside_a_compiled_function():
    """The calls break the graph and give what they give eagerly, gradients too."""
    ts = _scores()
    tokens = _tokens(37, 9001, 3).cuda()
    up = torch.randn(37, device="cuda")
    weight = torch.randn((900, 64), device="cuda").to(BF16)

    def step(x, hidden):
        got = ts.token_scores(x * 0.5, tokens, 5)
        head, entropy = ts.linear_token_scores(hidden + 1.0, weight, tokens % 900)
        return got.logprob * up + got.entropy + head - entropy, got.top_ids

    compiled = torch.compile(step, backend="aot_eager")
    results = []
    for run in (step, compiled):
        x = _logits(37, 9001, BF16, 3).cuda().requires_grad_(True)
        hidden = torch.ones((37, 64), device="cuda", dtype=BF16, requires_grad=True)
        score, ids = run(x, hidden)
        results.append([score, ids, *torch.autograd.grad(score.sum(), [x, hidden])])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 2, 255, 256, 257])
def test_parts_joined_by_several_lanes_and_by_one(rows):
    """Fewer rows than compute units join with several lanes on a key; both ways at top_k of
    powers of two and between."""
    ts = _scores()
    logits = (_logits(rows, 34000, F32, rows) * 4).round() / 4  # with ties
    tokens = _tokens(rows, 34000, rows)
    tokens[0] = 0
    x, t = logits.cuda(), tokens.cuda()
    ids = _top(logits, 64)
    want = _reference(logits, tokens, 1.0)[0]
    tol = _bounds(logits, 1.0)[0]
    for k in (1, 2, 3, 7, 8, 9, 31, 33, 63, 64):
        got = ts.token_scores(x, t, k)
        np.testing.assert_array_equal(got.top_ids.cpu().numpy(), ids[:, :k])
        _near(got.logprob, want, tol)


def test_python_launches_agree_with_the_native_ones(monkeypatch):
    from ops import _hip

    ts = _scores()
    assert _hip.host_ops() is not None
    logits, tokens = _logits(37, 9001, BF16, 3).cuda(), _tokens(37, 9001, 3).cuda()
    hidden = torch.randn((37, 60), generator=torch.Generator().manual_seed(1)).cuda()
    weight = torch.randn((9001, 60), generator=torch.Generator().manual_seed(2)).cuda()
    g, h = torch.randn(37, device="cuda"), torch.randn(37, device="cuda")

    def run():
        x = logits.clone().requires_grad_(True)
        got = ts.token_scores(x, tokens, 9, 0.9)
        grads = torch.autograd.grad([got.logprob, got.entropy], [x], [g, h])
        leaves = [hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)]
        scores = ts.linear_token_scores(*leaves, tokens, 0.9, 20)
        return (*got, *grads, *scores, *torch.autograd.grad(scores, leaves, [g, h]))

    native = run()
    monkeypatch.setattr(_hip, "host_ops", lambda: None)
    for a, b in zip(native, run()):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_second_derivatives_are_refused():
    ts = _scores()
    x = _logits(3, 50, F32, 3).cuda().requires_grad_(True)
    out = ts.token_scores(x, _tokens(3, 50, 3).cuda()).logprob.sum()
    with pytest.raises(RuntimeError, match="differentiate"):
        dx, = torch.autograd.grad(out, [x], create_graph=True)
        torch.autograd.grad(dx.sum(), [x])
    hidden = torch.randn((3, 16), device="cuda", requires_grad=True)
    weight = torch.randn((50, 16), device="cuda", requires_grad=True)
    out = ts.linear_token_scores(hidden, weight, _tokens(3, 50, 3).cuda())[0].sum()
    with pytest.raises(RuntimeError, match="differentiate"):
        dh, = torch.autograd.grad(out, [hidden], create_graph=True)
        torch.autograd.grad(dh.sum(), [hidden])


def test_a_changed_operand_is_noticed():
    ts = _scores()
    hidden = torch.randn((3, 16), device="cuda").to(BF16).requires_grad_(True)
    weight = torch.randn((50, 16), device="cuda").to(BF16).requires_grad_(True)
    out = ts.linear_token_scores(hidden, weight, torch.arange(3, device="cuda"))[0].sum()
    with torch.no_grad():
        weight.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, [hidden])


@pytest.mark.parametrize("native", [True, False])
def test_refusals_on_the_gpu(native, monkeypatch):
    """The same errors from either host path, before any launch."""
    from ops import _hip

    ts = _scores()
    if not native:
        monkeypatch.setattr(_hip, "host_ops", lambda: None)
    x, tokens = _logits(4, 30, F32, 1).cuda(), _tokens(4, 30, 1).cuda()
    cases = [((x.half(), tokens), "BF16 or FP32 logits"), ((x[0], tokens), "BF16 or FP32 logits"),
             ((x[:, :0], tokens), "1 to 524288"), ((x, tokens[:3]), "int64 vector"),
             ((x, tokens.int()), "int64 vector"), ((x, tokens.cpu()), "int64 vector"),
             ((x, tokens, 31), "top_k must lie"), ((x, tokens, -1), "top_k must lie"),
             ((torch.zeros((1, 524289), device="cuda"), tokens[:1]), "1 to 524288"),
             ((x, tokens, 1, 0.0), "temperature"), ((x, tokens, 1, float("nan")), "temperature")]
    for args, match in cases:
        with pytest.raises(ValueError, match=match):
            ts.token_scores(*args)
    h, w = torch.zeros((4, 16), device="cuda"), torch.zeros((30, 16), device="cuda")
    cases = [((h.half(), w, tokens), "BF16 or FP32"), ((h, w[:, :8], tokens), "Expected hidden"),
             ((h, w[:0], tokens), "Expected hidden"), ((h, w, tokens[:2]), "int64 vector"),
             ((h, w, tokens, -1.0), "temperature"), ((h, w, tokens, 1.0, 0), "chunk_rows")]
    for args, match in cases:
        with pytest.raises(ValueError, match=match):
            ts.linear_token_scores(*args)
