"""The table's gradient where it does not fit the caches, and past 2^31 elements, from sorted tokens some of which
are summed in pieces (GPU)."""
import pytest
import torch

from test_gpu_embedding import BF16, F32, F64, _check

pytestmark = pytest.mark.gpu


def _tokens(rows, vocab, seed):
    """Some from anywhere, the rest a few that occur more than 32 times, the table's last row among them; ignored
    and unknown ones between."""
    g = torch.Generator().manual_seed(seed)
    often = torch.tensor([vocab - 1, 0, vocab - 2, vocab // 2])
    t = torch.where(torch.rand(rows, generator=g) < 0.5, torch.randint(0, vocab, (rows,), generator=g),
                    often[torch.randint(0, 4, (rows,), generator=g)])
    t[3::29] = -100
    t[5::31] = vocab
    t[-40:] = vocab - 1
    assert torch.bincount(t[(t >= 0) & (t < vocab)]).max() > 32
    return t


def _check_rows(got, tokens, dy, vocab, scale, base=None):
    """The rows with tokens; all others are zeros (or, added to, what they were)."""
    known = (tokens >= 0) & (tokens < vocab)
    used, place = tokens[known].unique(return_inverse=True)
    small = torch.full_like(tokens, -100)
    small[known] = place
    used = used.cuda()
    _check(got[used], small, dy, len(used), scale, None if base is None else base[used])
    rest = torch.ones(vocab, dtype=torch.bool, device="cuda")
    rest[used] = False
    for part in torch.arange(vocab, device="cuda")[rest].split(1 << 18):
        assert not got[part].any() if base is None else torch.equal(got[part], base[part])


@pytest.mark.parametrize("dy_dtype", [BF16, F32])
@pytest.mark.parametrize("dtype,vocab", [(F32, 40000), (BF16, 70000)])
@pytest.mark.parametrize("rows", [100, 5000, 20000])
def test_past_the_caches(rows, dtype, vocab, dy_dtype):
    from ops.embedding_execution import embedding

    d = 2048
    assert vocab * d * dtype.itemsize > 256 << 20
    g = torch.Generator("cuda").manual_seed(rows)
    table = torch.randn((vocab, d), generator=g, device="cuda").to(dtype).requires_grad_(True)
    dy = torch.randn((rows, d), generator=g, device="cuda").to(dy_dtype)
    tokens = _tokens(rows, vocab, seed=rows)
    device_tokens = tokens.cuda()
    got, = torch.autograd.grad(embedding(device_tokens, table, 0.75, dy_dtype), [table], dy)
    _check_rows(got, tokens, dy, vocab, 0.75)
    again, = torch.autograd.grad(embedding(device_tokens, table, 0.75, dy_dtype), [table], dy)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,d", [(300, 2048), (300, 2047), (9000, 2048)])
def test_sorted_past_2_31_elements(rows, d, dtype):
    from ops.embedding_execution import embedding

    vocab = 1050000
    assert (vocab - 1) * d > 2 ** 31
    g = torch.Generator("cuda").manual_seed(rows + d)
    table = torch.zeros((vocab, d), dtype=dtype, device="cuda").requires_grad_(True)
    dy = torch.randn((rows, d), generator=g, device="cuda").to(BF16)
    tokens = _tokens(rows, vocab, seed=d)
    got, = torch.autograd.grad(embedding(tokens.cuda(), table, -2.0), [table], dy)
    _check_rows(got, tokens, dy, vocab, -2.0)


@pytest.mark.parametrize("rows,d", [(40, 2048), (300, 2048), (300, 2047)])
def test_added_past_2_31_elements(rows, d):
    from ops.embedding_execution import embedding_accumulate_

    vocab = 1050000
    g = torch.Generator("cuda").manual_seed(rows + d)
    base = torch.randn((vocab, d), generator=g, device="cuda")
    dy = torch.randn((rows, d), generator=g, device="cuda").to(BF16)
    tokens = _tokens(rows, vocab, seed=d)
    _check_rows(embedding_accumulate_(base.clone(), tokens.cuda(), dy, 0.5), tokens, dy, vocab, 0.5, base)
