"""Token scores of logits of any finite size: masks of the type's lowest value, offsets whose
rounding is larger than the logits' differences, and certain tokens (GPU, against 64 bits)."""
import math

import pytest
import torch

from test_gpu_token_scores import BF16, F32, F64, U, _reference, _top

pytestmark = pytest.mark.gpu


def _scores():
    from ops import token_scores

    return token_scores


def _bounds(logits, temperature):
    """(lse and log probability, entropy, probability) bounds as test_gpu_token_scores._bounds has
    them, but of the logits' distances to their row's largest, as far as e^-distance is no zero
    in FP32 (distances up to 110 temperatures): arithmetic on the distances rounds nothing else."""
    wide = logits.to(F64)
    far = (wide.amax(-1, keepdim=True) - wide) / temperature
    near = far[far < 110.0]
    r = float(near.max()) + math.log(logits.shape[1])
    rel = (3 * r + 2) * 2 * U + 64 * U
    score = rel + 8 * r * U
    return score, (1 + 2 * r) * 2 * rel + 8 * r * U, rel


def _near(got, want, tol):
    """Within tol and four roundings of the value's own size (the distance, times 1 / temperature,
    itself rounded, and the logarithm taken off); beyond FP32's range infinite."""
    got, want = got.detach().double().cpu(), want.double()
    narrow = want.float().double()
    assert torch.equal(torch.isfinite(got), torch.isfinite(narrow)) and not bool(torch.isnan(got).any())
    finite = torch.isfinite(narrow)
    assert torch.equal(got[~finite], narrow[~finite])
    ratio = ((got - want).abs() / (tol + 4 * U * want.abs()))[finite]
    assert bool((ratio <= 1.0).all()), float(ratio.max())


def _random(rows, vocab, dtype, seed, std=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g) * std).to(dtype)


def _masked(name, rows, vocab, dtype):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = _random(rows, vocab, dtype, vocab)
    if name == "every":
        x[::2] = low
    elif name == "some":
        x[:, torch.arange(vocab) % 3 != 1] = low
    elif name == "most":  # fewer tokens left than are asked for
        x[:, torch.arange(vocab) >= 5] = low
    elif name == "with -inf":
        x[:, torch.arange(vocab) % 3 != 1] = low
        x[::2, torch.arange(vocab) % 3 == 1] = -float("inf")
        x[:, ::5] = -float("inf")
    elif name == "one highest":
        x[:, vocab // 2] = high
    elif name == "all highest":
        x[:] = high
    return x


MASKS = ["every", "some", "most", "with -inf", "one highest", "all highest"]
# One part a row, several parts, the most parts, and parts of 2048 for few rows.
SIZES = [(3, 7), (5, 300), (300, 9001), (2, 40000), (1, 524288)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 1.3])
@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("name", MASKS)
def test_finite_masks(name, rows, vocab, temperature, dtype):
    """The masked tokens have probability zero in a row with others and share it in a row without,
    and a masked token's own score is its distance."""
    ts = _scores()
    x = _masked(name, rows, vocab, dtype)
    score_tol, entropy_tol, _ = _bounds(x, temperature)
    k = min(vocab, 8)
    ids = torch.from_numpy(_top(x, k))
    for column in (0, vocab // 2, vocab - 1):
        tokens = torch.full((rows,), column)
        logprob, entropy, logp, _ = _reference(x, tokens, temperature)
        got = ts.token_scores(x.cuda(), tokens.cuda(), k, temperature)
        _near(got.logprob, logprob, score_tol)
        _near(got.entropy, entropy, entropy_tol)
        assert torch.equal(got.top_ids.cpu(), ids)
        _near(got.top_logprobs, logp.gather(1, ids), score_tol)


def _offset(rows, vocab, offset, step):
    """offset + j step, j = 0 .. 5: FP32 numbers whose distances are exact."""
    j = torch.randint(0, 6, (rows, vocab), generator=torch.Generator().manual_seed(vocab)).double()
    wide = offset + step * j
    assert torch.equal(wide.float().double(), wide)
    return wide.float()


# An offset, and the step by which FP32 numbers near it differ (a temperature, too).
OFFSETS = [(1000.0, 2.0 ** -10), (-1e9, 64.0), (1e10, 1024.0), (-(2.0 ** 100), 2.0 ** 77), (2.0 ** 127, 2.0 ** 104)]


@pytest.mark.parametrize("offset,step", OFFSETS)
@pytest.mark.parametrize("rows,vocab", [(3, 300), (300, 9001), (1, 40000)])
def test_far_from_zero(rows, vocab, offset, step):
    """Only the distances count: scores and gradients are those of the logits without their
    offset."""
    ts = _scores()
    x, small = _offset(rows, vocab, offset, step), _offset(rows, vocab, 0.0, 1.0)
    tokens = torch.arange(rows) % vocab
    g, h = torch.linspace(-1, 1, rows), torch.linspace(0.5, -0.7, rows)
    logprob, entropy, _, grad = _reference(small, tokens, 1.0, g, h)
    score_tol, entropy_tol, _ = _bounds(small, 1.0)
    leaf = x.cuda().requires_grad_(True)
    got = ts.token_scores(leaf, tokens.cuda(), 4, step)
    _near(got.logprob, logprob, score_tol)
    _near(got.entropy, entropy, entropy_tol)
    assert torch.equal(got.top_ids.cpu(), torch.from_numpy(_top(small, 4)))
    dx, = torch.autograd.grad([got.logprob, got.entropy], [leaf], [g.cuda(), h.cuda()])
    # (A power of two: the gradient times it is that of the distances.)
    _check_gradient(dx.double() * step, F32, grad, small, tokens, g, h, 1.0)


def _check_gradient(dx, dtype, want, x, tokens, g, h, temperature):
    """The bound of test_gpu_token_scores.test_gradient_of_the_logits: every factor's own error.
    (A probability below FP32's normal numbers may be taken as zero: less than 1e-30.)"""
    score_tol, entropy_tol, rel = _bounds(x, temperature)
    _, entropy, logp, _ = _reference(x, tokens, temperature)
    p = logp.exp()
    surprise = torch.where(p > 0, logp.abs(), torch.zeros_like(p)) + entropy[:, None]
    size = p * (g.abs()[:, None] + h.abs()[:, None] * surprise) / temperature
    bound = size * (rel + score_tol + 16 * U) + p * h.abs()[:, None] * (score_tol + entropy_tol) / temperature
    bound = bound + (torch.finfo(dtype).eps / 2 + 4 * U) * (want.abs() + bound) + 1e-30
    worst = float(((dx.double().cpu() - want).abs() / bound).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 1.3])
@pytest.mark.parametrize("rows,vocab", [(3, 7), (5, 300), (40, 9001), (1, 40000)])
@pytest.mark.parametrize("name", MASKS)
def test_gradients_of_finite_masks(name, rows, vocab, temperature, dtype):
    ts = _scores()
    x = _masked(name, rows, vocab, dtype)
    tokens = torch.arange(rows) * 3 % vocab
    tokens[-1] = -100
    g, h = torch.linspace(-1, 1, rows), torch.linspace(0.5, -0.7, rows)
    want = _reference(x, tokens, temperature, g, h)[3]
    leaf = x.cuda().requires_grad_(True)
    got = ts.token_scores(leaf, tokens.cuda(), 0, temperature)
    dx, = torch.autograd.grad([got.logprob, got.entropy], [leaf], [g.cuda(), h.cuda()])
    assert dx.dtype == dtype
    _check_gradient(dx, dtype, want, x, tokens, g, h, temperature)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("value", [19.875, 30.3, 999.7, -1000.9, 3e30])
def test_certain_tokens(value, dtype):
    """A log probability is at most zero: of a vocabulary of one, and of a token far above the
    others (at least 19.8 for each)."""
    ts = _scores()
    one = torch.full((2, 1), value).to(dtype).cuda()
    got = ts.token_scores(one, torch.zeros(2, dtype=torch.int64, device="cuda"), 1, 0.9)
    for t in (got.logprob, got.entropy, got.top_logprobs):
        assert not bool(t.any())
    for rows, vocab in ((2, 200), (300, 9001)):
        x = torch.full((rows, vocab), value).to(dtype)
        x -= x.abs() * torch.rand((rows, vocab), generator=torch.Generator().manual_seed(1)).to(dtype).clamp(0, 0.1)
        x -= x.abs()
        x[:, 77] = torch.tensor(value).to(dtype)
        tokens = torch.full((rows,), 77)
        logprob, entropy, _, _ = _reference(x, tokens, 1.0)
        got = ts.token_scores(x.cuda(), tokens.cuda(), 1)
        assert bool((got.logprob <= 0.0).all()) and torch.equal(got.logprob, got.top_logprobs[:, 0])
        # At most 64 additions beside the 1, and each term's own relative error (_bounds at a
        # distance of 29: 242 U, and the logarithm's); distances beyond that add nothing.
        for out, want in ((got.logprob, logprob), (got.entropy, entropy)):
            assert bool(((out.cpu().double() - want).abs() <= 72 * U + 300 * U * want.abs()).all())


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("rows,vocab", [(5, 300), (300, 2056), (2100, 264)])
def test_head_logits_of_any_size(rows, vocab, sign):
    """hidden @ weight.T with one column that makes every logit 1.75 2^127 and others that are
    exact beside it: a uniform distribution, and half the vocabulary at 0."""
    ts = _scores()
    hidden, weight = torch.zeros((rows, 16)), torch.zeros((vocab, 16))
    hidden[:, 0], weight[:, 0] = 2.0 ** 63, sign * 1.75 * 2.0 ** 64
    tokens = torch.arange(rows) % vocab
    for low in (False, True):
        if low:
            weight[vocab // 2:, 0] = 0.0
        logits = hidden.double() @ weight.double().T
        logprob, entropy, _, _ = _reference(logits, tokens, 1.0)
        # FP32 sums of equal terms (counts): the logarithm's and the final roundings.
        got = ts.linear_token_scores(hidden.to(BF16).cuda(), weight.to(BF16).cuda(), tokens.cuda())
        _near(got[0], logprob, 64 * U * math.log(vocab))
        _near(got[1], entropy, 64 * U * math.log(vocab))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradient_over_the_logits(dtype):
    """The C entry point's gradient in place of the logits, of rows of every kind: as beside them."""
    from ops import _hip

    ts = _scores()
    rows, vocab = 40, 9001
    x = _masked("every", rows, vocab, dtype)
    x[1::4] = _random(10, vocab, dtype, 1).add_(3000.0)
    x = x.cuda().requires_grad_(True)
    tokens = torch.arange(rows).cuda()
    g, h = torch.linspace(-1, 1, rows).cuda(), torch.linspace(0.5, -0.7, rows).cuda()
    got = ts.token_scores(x, tokens)
    want, = torch.autograd.grad([got.logprob, got.entropy], [x], [g, h])
    inplace = x.detach().clone()
    lse, logprob, entropy = torch.empty((3, rows), device="cuda").unbind()
    need = _hip.query_on(inplace, "ws_token_scores_workspace_bytes", rows, vocab, 0)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    _hip.call_on(inplace, "ws_token_scores", inplace.data_ptr(), vocab, int(dtype == F32), tokens.data_ptr(), rows,
                 vocab, 1.0, 0, work.data_ptr(), lse.data_ptr(), logprob.data_ptr(), entropy.data_ptr(), None, None)
    _hip.call_on(inplace, "ws_token_scores_backward", inplace.data_ptr(), vocab, int(dtype == F32),
                 tokens.data_ptr(), rows, vocab, 1.0, lse.data_ptr(), entropy.data_ptr(), g.data_ptr(),
                 h.data_ptr(), inplace.data_ptr(), vocab)
    assert torch.equal(inplace, want) and bool(inplace.any())
