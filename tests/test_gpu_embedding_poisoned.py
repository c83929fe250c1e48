"""The gradient of an embedding into memory that held NaN before: every element of dW is written and finite, rows that no token
names are zero, in each of the ways the gradient is computed.  Beside the tolerance of test_gpu_embedding a comparison that a
NaN does not pass."""
import pytest
import torch

import elixir_amd as ea

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def poison(*sizes):
    """Leaves blocks of these sizes full of NaN to the allocator: what is allocated next, of such a size, takes them."""
    blocks = [torch.full((n, ), 0xFF, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(3)]
    del blocks


def gradient(index, table, dy, padding_idx, scale):
    y = ea.embedding(index, table, padding_idx=padding_idx, scale=scale)
    poison(y.numel() * table.element_size(), 1 << 16, 1 << 22)    # a workspace, for one
    poison(table.numel() * table.element_size())    # dW, the first that backward allocates
    assert not torch.isfinite(torch.empty_like(table)).any()
    return torch.autograd.grad(y, table, dy)[0]


def verify(got, index, table, dy, padding_idx, scale):
    flat = index.reshape(-1).long()
    g = dy.double().reshape(flat.numel(), table.shape[1])
    keep = (flat >= 0) & (flat < table.shape[0])
    if padding_idx is not None:
        keep &= flat != padding_idx
    g, at = g[keep], flat[keep]
    want = torch.zeros(table.shape, dtype=torch.float64, device=DEV).index_add_(0, at, g) * scale
    size = torch.zeros(table.shape, dtype=torch.float64, device=DEV).index_add_(0, at, g.abs()) * abs(scale)
    count = torch.bincount(at, minlength=table.shape[0])[:, None]
    tiny = torch.finfo(table.dtype).tiny if table.dtype == torch.float16 else 0.0
    tol = 2.0**-24 * (count + 2) * size + torch.finfo(table.dtype).eps / 2 * want.abs().clamp_min(tiny) * (count > 0)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f'{int(bad.sum())} elements'
    assert not got[count[:, 0] == 0].any()


# few tokens in one launch; the sort of one workgroup; the sort of many and its join, short tiles and long ones; each with rows that
# are moved 16 bytes at a time and element by element, and tables far longer than the batch
CASES = [(1, 1000, 64), (7, 50257, 96), (1000, 5000, 65), (1024, 50257, 768), (1023, 33, 4100), (1025, 3000, 64), (2048, 700, 771),
         (2049, 50272, 64), (5000, 10, 1000), (8192, 30000, 33), (9000, 4000, 2048), (20000, 1000, 1025), (70000, 2, 256), (3000, 20000, 1)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tokens,vocab,cols', CASES)
def test_every_element_is_written(tokens, vocab, cols, dtype):
    g = torch.Generator(device=DEV).manual_seed(tokens)
    index = (torch.rand(tokens, generator=g, device=DEV)**3 * vocab).long().clamp_(max=vocab - 1)
    table = torch.zeros(vocab, cols, dtype=dtype, device=DEV).requires_grad_()
    dy = torch.randn(tokens, cols, generator=g, device=DEV).to(dtype)
    verify(gradient(index, table, dy, None, 1.5), index, table.detach(), dy, None, 1.5)


@pytest.mark.parametrize('tokens,cols', [(300, 64), (1500, 65), (4000, 512)])
@pytest.mark.parametrize('kind', ['all padding', 'all outside', 'half outside', 'one index', 'last row'])
def test_batches_that_name_few_rows(tokens, cols, kind):
    vocab = 3000
    g = torch.Generator(device=DEV).manual_seed(cols)
    index = torch.randint(0, vocab, (tokens, ), generator=g, device=DEV)
    padding = None
    if kind == 'all padding':
        index.fill_(17)
        padding = 17
    elif kind == 'all outside':
        index += vocab
        index[::2] *= -1
    elif kind == 'half outside':
        index[::2] = -1 - index[::2]
    elif kind == 'one index':
        index.fill_(vocab // 2)
    else:
        index.fill_(vocab - 1)
    table = torch.zeros(vocab, cols, dtype=torch.bfloat16, device=DEV).requires_grad_()
    dy = torch.randn(tokens, cols, generator=g, device=DEV).bfloat16()
    verify(gradient(index, table, dy, padding, 1.0), index, table.detach(), dy, padding, 1.0)


def test_the_comparison_sees_a_row_that_is_not_written():
    """The mistake planted in what the comparison is given."""
    index, table = torch.tensor([1, 2], device=DEV), torch.zeros(4, 8, device=DEV)
    dy = torch.ones(2, 8, device=DEV)
    good = torch.zeros(4, 8, device=DEV)
    good[1:3] = 1
    verify(good, index, table, dy, None, 1.0)
    for row in (0, 1):
        bad = good.clone()
        bad[row, 3] = float('nan')
        with pytest.raises(AssertionError):
            verify(bad, index, table, dy, None, 1.0)
