"""Embedding lookup and the table's gradient against plain sums in 64 bits (GPU).

The lookup is one FP32 product, rounded: its bits are PyTorch's. A gradient of n FP32 terms is off by at
most n 2^-24 of their magnitudes, plus half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24


def _tokens(rows, vocab, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((rows,), vocab // 2)
    if kind == "zipf":
        return ((vocab + 1.0) ** torch.rand((rows,), generator=g, dtype=F64)).long().sub_(1).clamp_(0, vocab - 1)
    if kind == "runs":  # a few tokens, in long runs
        return (torch.arange(rows) // 97 * 31) % min(vocab, 5)
    t = torch.randint(0, vocab, (rows,), generator=g)
    if kind == "ignored":
        t[torch.rand((rows,), generator=g) < 0.3] = -100
        t[::13] = vocab
        t[5::17] = -1
        t[7::19] = 2 ** 40
    return t


def _check(got, tokens, dy, vocab, scale, base=None):
    known = (tokens >= 0) & (tokens < vocab)
    t, g = tokens[known].cuda(), dy.reshape(-1, dy.shape[-1])[known.cuda()].to(F64)
    want = torch.zeros((vocab, dy.shape[-1]), dtype=F64, device="cuda").index_add_(0, t, g * scale)
    size = torch.zeros_like(want).index_add_(0, t, g.abs() * abs(scale))
    n = torch.bincount(t, minlength=vocab)[:, None]
    if base is not None:
        want, size = want + base.to(F64), size + base.to(F64).abs()
    bound = (n + 3) * U * size + want.abs() * torch.finfo(got.dtype).eps / 2
    off = (got.to(F64) - want).abs()
    assert got.isfinite().all() and (off <= bound).all(), (off / bound.clamp_min(1e-300)).max().item()


@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("table_dtype", [BF16, F32])
@pytest.mark.parametrize("rows,vocab,d", [(1, 1, 1), (1, 300, 2048), (48, 1000, 1280), (37, 50, 77),
                                          (5, 9, 8200), (4100, 777, 136)])
def test_lookup(rows, vocab, d, table_dtype, out):
    from ops.embedding_execution import embedding

    table = torch.randn((vocab, d), generator=torch.Generator().manual_seed(d)).to(table_dtype).cuda()
    tokens = _tokens(rows, vocab, "ignored", seed=rows).cuda()
    for scale in (1.0, 0.3, -35.777):
        got = embedding(tokens, table, scale, out)
        known = (tokens >= 0) & (tokens < vocab)
        want = (table[tokens.clamp(0, vocab - 1)].float() * scale).to(out)
        assert got.dtype == out and torch.equal(got[known], want[known])
        assert not got[tokens == -100].any()
        assert got[~known & (tokens != -100)].isnan().all()


@pytest.mark.parametrize("kind", ["any", "one", "zipf", "runs", "ignored"])
@pytest.mark.parametrize("rows,vocab,d,table_dtype,out", [
    (1, 1, 1, F32, BF16), (31, 7, 64, BF16, BF16), (32, 600, 512, F32, BF16), (33, 40, 77, BF16, BF16),
    (64, 9, 2100, F32, F32), (64, 333, 4104, BF16, BF16), (65, 9, 2100, F32, BF16),
    (1000, 3000, 1280, BF16, F32), (1025, 511, 2048, F32, F32), (2500, 97, 1001, F32, BF16),
    (5000, 140001, 24, F32, BF16), (40000, 5000, 256, F32, BF16), (40001, 300, 2056, BF16, BF16),
    (70, 5001, 136, F32, BF16)])
def test_gradient(rows, vocab, d, table_dtype, out, kind):
    from ops.embedding_execution import embedding

    g = torch.Generator().manual_seed(rows + vocab + d)
    table = torch.randn((vocab, d), generator=g).to(table_dtype).cuda().requires_grad_(True)
    dy = torch.randn((rows, d), generator=g).to(out).cuda()
    tokens = _tokens(rows, vocab, kind, seed=d)
    scale = 0.75 if rows % 2 else 1.0
    y = embedding(tokens.cuda(), table, scale, out)
    got, = torch.autograd.grad(y, [table], dy)
    assert got.dtype == table_dtype and got.shape == table.shape
    _check(got, tokens, dy, vocab, scale)
    again, = torch.autograd.grad(embedding(tokens.cuda(), table, scale, out), [table], dy)
    assert torch.equal(got, again)


@pytest.mark.parametrize("kind", ["one", "zipf", "ignored"])
@pytest.mark.parametrize("rows,vocab,d,dtype", [(1, 20, 8, BF16), (50, 30, 2050, F32), (700, 4000, 640, BF16), (3000, 50, 333, F32),
                                                (9000, 12000, 128, BF16)])
def test_accumulate(rows, vocab, d, dtype, kind):
    from ops.embedding_execution import embedding_accumulate_

    g = torch.Generator().manual_seed(rows)
    base = torch.randn((vocab, d + 5), generator=g).cuda()
    tokens = _tokens(rows, vocab, kind, seed=3)
    dy = torch.randn((rows, d), generator=g).to(dtype).cuda()
    used = torch.zeros(vocab, dtype=torch.bool)
    used[tokens[(tokens >= 0) & (tokens < vocab)]] = True
    # Rows without tokens, and columns beside the gradient, are left as they were.
    for columns in (slice(0, d), slice(4, 4 + d), slice(5, 5 + d)):
        wide = base.clone()
        wide[~used.cuda()] = float("nan")
        before = wide.clone()
        out = wide[:, columns]
        version = wide._version
        assert embedding_accumulate_(out, tokens.cuda(), dy, 0.5) is out and wide._version > version
        _check(out[used.cuda()], torch.cumsum(used, 0)[tokens.clamp(0, vocab - 1)].sub(1).masked_fill(
            (tokens < 0) | (tokens >= vocab), -100), dy, int(used.sum()), 0.5,
            before[:, columns][used.cuda()])
        assert out[~used.cuda()].isnan().all()
        rest = torch.ones(d + 5, dtype=torch.bool)
        rest[columns] = False
        assert torch.equal(wide[:, rest.cuda()][used.cuda()], before[:, rest.cuda()][used.cuda()])


def test_joins_a_tied_heads_gradient():
    from ops.embedding_execution import embedding, embedding_accumulate_

    g = torch.Generator().manual_seed(5)
    table = torch.randn((500, 96), generator=g).cuda().requires_grad_(True)
    tokens = _tokens(300, 500, "zipf").cuda()
    dy = torch.randn((300, 96), generator=g).to(BF16).cuda()
    head = torch.randn((500, 96), generator=g).cuda()
    d, = torch.autograd.grad(embedding(tokens, table, 2.0), [table], dy)
    assert torch.equal(embedding_accumulate_(head.clone(), tokens, dy, 2.0), head + d)


def test_empty_and_shaped_tokens():
    from ops.embedding_execution import embedding, embedding_accumulate_

    table = torch.randn((40, 64), device="cuda").requires_grad_(True)
    none = torch.zeros((0,), dtype=torch.int64, device="cuda")
    y = embedding(none, table)
    assert y.shape == (0, 64)
    assert not torch.autograd.grad(y.sum(), [table])[0].any()
    grad = torch.ones((40, 64), device="cuda")
    assert torch.equal(embedding_accumulate_(grad, none, y.detach()), torch.ones_like(grad))
    tokens = torch.arange(24, device="cuda").view(2, 3, 4)
    y = embedding(tokens.transpose(0, 2), table)
    assert torch.equal(y, table.detach()[tokens.transpose(0, 2)].to(BF16))
    d, = torch.autograd.grad(y.sum(), [table])
    assert (d[:24] == 1).all() and not d[24:].any()
    scalar = embedding(torch.tensor(3, device="cuda"), table)
    assert torch.equal(scalar, table.detach()[3].to(BF16))


def test_table_layouts():
    from ops.embedding_execution import embedding

    base = torch.randn((50, 70), device="cuda").to(BF16)
    tokens = _tokens(33, 50, "any").cuda()
    for table in (base[:, 3:67], base[:, :64], base.t().contiguous().t()[:, :64], base[::2]):
        leaf = table.detach().requires_grad_(True)
        t = tokens % table.shape[0]
        y = embedding(t, leaf)
        assert torch.equal(y, table[t])
        d, = torch.autograd.grad(y.sum(), [leaf])
        assert torch.equal(d, torch.bincount(t, minlength=len(table))[:, None].expand_as(table).to(BF16))


def test_python_form_gives_the_same_bits(monkeypatch):
    from ops import _hip
    from ops.embedding_execution import embedding, embedding_accumulate_

    def run():
        g = torch.Generator().manual_seed(1)
        table = torch.randn((700, 130), generator=g).cuda().requires_grad_(True)
        tokens = _tokens(2000, 700, "zipf").cuda()
        dy = torch.randn((2000, 130), generator=g).to(BF16).cuda()
        y = embedding(tokens, table, 0.5)
        d, = torch.autograd.grad(y, [table], dy)
        return y, d, embedding_accumulate_(torch.ones((700, 130), device="cuda"), tokens, dy)

    want = run()
    monkeypatch.setattr(_hip, "host_ops", lambda: None)
    for a, b in zip(run(), want):
        assert torch.equal(a, b)


def test_past_2_31_elements():
    from ops.embedding_execution import embedding

    vocab, d = 1050000, 2048
    table = torch.zeros((vocab, d), dtype=BF16, device="cuda")
    table[-3:] = torch.randn((3, d), device="cuda").to(BF16)
    table.requires_grad_(True)
    tokens = torch.tensor([vocab - 1, 0, vocab - 3, vocab - 1], device="cuda")
    y = embedding(tokens, table, 2.0)
    assert torch.equal(y, (table.detach()[tokens].float() * 2).to(BF16))
    dy = torch.randn((4, d), device="cuda").to(BF16)
    got, = torch.autograd.grad(y, [table], dy)
    assert torch.equal(got[vocab - 1], ((dy[0].float() + dy[3].float()) * 2).to(BF16))
    assert torch.equal(got[vocab - 3], (dy[2].float() * 2).to(BF16))
    assert torch.equal(got[0], (dy[1].float() * 2).to(BF16))
    assert not got[1:vocab - 3].any() and not got[vocab - 2].any()
