"""embedding on the GPU: forward bit for bit, the gradient of the table against float64.

Tolerance of a gradient, derived beforehand: a row that `count` tokens name is a sum of `count` fp32 numbers in some fixed
order, `count` roundings at most on the way of each (2^-24 of the partial sums, which sum |dy| bounds), one for the scale, and
half a step of the type at the end: 2^-24 (count + 2) |scale| sum |dy| + half a step."""
import pytest
import torch

import elixir_amd as ea

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dtype, ref):
    return torch.finfo(dtype).eps / 2 * ref.abs().clamp_min(torch.finfo(dtype).tiny if dtype == torch.float16 else 0.0)


def run(index, table, dy, **kw):
    table.requires_grad_()
    y = ea.embedding(index, table, **kw)
    return y, torch.autograd.grad(y, table, dy)[0]


def check(index, table, dy, padding_idx=None, scale=1.0):
    y, dtable = run(index, table, dy, padding_idx=padding_idx, scale=scale)
    flat = index.reshape(-1).long()
    assert y.shape == index.shape + table.shape[1:]
    with torch.no_grad():
        assert torch.equal(y, (table.detach()[flat].float() * torch.tensor(scale, dtype=torch.float32)).to(table.dtype).view(y.shape))
    g = dy.double().reshape(flat.numel(), table.shape[1])
    keep = flat >= 0
    if padding_idx is not None:
        keep &= flat != padding_idx % table.shape[0]
    g, at = g[keep], flat[keep]
    want = torch.zeros(table.shape, dtype=torch.float64, device=DEV).index_add_(0, at, g) * scale
    size = torch.zeros(table.shape, dtype=torch.float64, device=DEV).index_add_(0, at, g.abs()) * abs(scale)
    count = torch.bincount(at, minlength=table.shape[0])[:, None]
    tol = 2.0**-24 * (count + 2) * size + half_step(table.dtype, want) * (count > 0)
    bad = (dtable.double() - want).abs() > tol
    assert not bad.any(), f'{int(bad.sum())} elements, worst {(dtable.double() - want).abs().max().item():.3g}'
    return dtable


def make(tokens, vocab, cols, dtype, seed=0, skew=3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    index = (torch.rand(tokens, generator=g, device=DEV)**skew * vocab).long().clamp_(max=vocab - 1)
    return (index, torch.randn(vocab, cols, generator=g, device=DEV).to(dtype), torch.randn(tokens, cols, generator=g, device=DEV).to(dtype))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('cols', [1, 3, 4, 7, 8, 16, 64, 100, 256, 257, 512, 520, 769, 1024, 2048, 2056, 5000])
def test_every_width(cols, dtype):
    check(*make(301, 97, cols, dtype, seed=cols), scale=1.5)


@pytest.mark.parametrize('tokens', [1, 2, 31, 32, 33, 63, 64, 65, 1023, 1024, 1025, 4097, 70001])
@pytest.mark.parametrize('vocab', [1, 2, 10, 1023, 1024, 1025, 50257])
def test_tokens_and_vocabularies(tokens, vocab):
    """Runs that end inside a tile, at its end and tiles later; one to three passes of the sort; one and more rounds and
    workgroups of it."""
    check(*make(tokens, vocab, 24, torch.float32, seed=tokens + vocab))
    check(*make(tokens, vocab, 5, torch.bfloat16, seed=tokens + vocab, skew=1))


def test_three_passes_of_the_sort():
    check(*make(3000, (1 << 20) + 77, 8, torch.float16, skew=1))
    index, table, dy = make(3000, (1 << 20) + 77, 8, torch.float16, skew=1)
    index[:] = torch.randint(0, 40, (3000, ), device=DEV) * 26215
    check(index, table, dy)


@pytest.mark.parametrize('dtype', DTYPES)
def test_one_token_fills_the_batch(dtype):
    index, table, dy = make(20000, 1000, 136, dtype)
    index.fill_(999)
    check(index, table, dy)
    index[7000:7033] = 0
    index[0], index[-1] = 5, 998
    d = check(index, table, dy, scale=0.25)
    assert torch.equal(d, run(index, table, dy, scale=0.25)[1])    # the same bits again


@pytest.mark.parametrize('padding_idx', [0, 3, -1, 999])
def test_padding(padding_idx):
    index, table, dy = make(5000, 1000, 72, torch.float16)
    index[1000:3000] = padding_idx % 1000
    d = check(index, table, dy, padding_idx=padding_idx)
    assert not d[padding_idx].any()
    index.fill_(padding_idx % 1000)
    assert not run(index, table, dy, padding_idx=padding_idx)[1].any()


def test_types_shapes_and_strides_of_the_indices():
    index, table, dy = make(600, 50, 40, torch.float32)
    for idx in (index.int(), index.view(3, 200), index.view(20, 30).t(), index[::2], index[:1].view(()), index.view(2, 300)[:, :7],
                index[:1].expand(9)):
        check(idx, table, torch.randn(*idx.shape, 40, device=DEV))
    check(index, torch.randn(50, 41, device=DEV)[:, 1:], dy)                      # a table that is a slice
    check(index, table, torch.randn(600, 1, device=DEV).expand(600, 40))          # gradients that arrive expanded
    wide = torch.randn(600, 48, device=DEV)
    check(index, table, wide[:, :40])                                             # rows apart, read in place
    check(index, table, wide[:, 3:43])
    big = torch.zeros(50 * 40 + 1, device=DEV)[1:].view(50, 40)                   # a table at an odd address
    big.copy_(table.detach())
    check(index, big, dy)


def test_indices_outside_the_table():
    """A row of NaN and no gradient; nothing is read or written outside."""
    index, table, dy = make(300, 50, 40, torch.float32)
    good = index.clone()
    index[5], index[77], index[299] = -1, 50, 1 << 40
    y, d = run(index, table, dy)
    bad = [5, 77, 299]
    keep = torch.ones(300, dtype=torch.bool, device=DEV)
    keep[bad] = False
    assert torch.isnan(y[bad]).all() and torch.equal(y[keep], table.detach()[good[keep]])
    masked = dy.clone()
    masked[bad] = 0
    want = run(good, table, masked)[1]
    torch.testing.assert_close(d, want, rtol=1e-5, atol=1e-5)
    y = ea.embedding(torch.full((3, ), -1, dtype=torch.int32, device=DEV), table.detach())
    assert torch.isnan(y).all()


def test_gradients_that_are_not_finite_stay_in_their_rows():
    index, table, dy = make(2000, 100, 16, torch.float32)
    dy[3, 5], dy[700, 0] = float('inf'), float('nan')
    d = run(index, table, dy)[1]
    hit = torch.zeros(100, 16, dtype=torch.bool, device=DEV)
    hit[index[3], 5] = hit[index[700], 0] = True
    assert torch.equal(~torch.isfinite(d), hit)


def test_empty():
    table = torch.randn(10, 4, device=DEV)
    y, d = run(torch.zeros(0, 3, dtype=torch.int64, device=DEV), table, torch.zeros(0, 3, 4, device=DEV))
    assert y.shape == (0, 3, 4) and not d.any()
    assert ea.embedding(torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(10, 0, device=DEV)).shape == (2, 0)


def test_refusals_on_device_tensors():
    index, table, _ = make(4, 10, 8, torch.float32)
    with pytest.raises(TypeError, match='float64'):
        ea.embedding(index, table.double())
    with pytest.raises(RuntimeError, match='GPU'):
        ea.embedding(index.cpu(), table)
    with pytest.raises(ValueError, match='padding_idx'):
        ea.embedding(index, table, padding_idx=10)
    with pytest.raises(ValueError, match='table of 1'):
        ea.embedding(index, table[:0])


def test_a_gradient_can_be_differentiated():
    out = []
    for f in (lambda i, t: ea.embedding(i, t, padding_idx=2, scale=3.0), lambda i, t: torch.nn.functional.embedding(i, t, padding_idx=2) * 3):
        index, table, _ = make(50, 10, 8, torch.float32)
        table.requires_grad_()
        g, = torch.autograd.grad(f(index, table).pow(3).sum(), table, create_graph=True)
        out.append((g, torch.autograd.grad(g.square().sum(), table)[0]))
    for got, want in zip(*out):
        torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5 * want.abs().max().item())


def test_gradient_against_differences():
    """sum(c y) is linear in the table: a difference along d is scale * sum(c d[index]), whatever the step."""
    index, table, c = make(700, 90, 33, torch.float32)
    d = torch.randn(90, 33, device=DEV).mul(16).round() / 16
    base = torch.randn(90, 33, device=DEV).mul(16).round() / 16    # sums and differences of these are exact
    grad = run(index, base, c, scale=2.0)[1].double()
    diff = ((ea.embedding(index, base.detach() + d, scale=2.0).double() - ea.embedding(index, base.detach() - d, scale=2.0).double())
            * c.double()).sum() / 2
    size = (c.double().abs() * d.double().abs()[index]).sum()
    assert (diff - (grad * d.double()).sum()).abs() <= 2.0**-24 * 702 * 2 * size


def test_streams_and_graphs():
    index, table, dy = make(3000, 500, 128, torch.bfloat16)
    want = run(index, table, dy, scale=3.0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            results.append(run(index, table.detach().clone(), dy, scale=3.0))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, e) for a, e in zip(r, want))
    del want, results
    si, st, sg = index.clone(), table.detach().clone(), dy.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(si, st, sg, scale=3.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(si, st, sg, scale=3.0)
    for seed in range(1, 5):
        ni, nt, ng = make(3000, 500, 128, torch.bfloat16, seed=seed, skew=seed)
        with torch.no_grad():
            si.copy_(ni), st.copy_(nt), sg.copy_(ng)
        graph.replay()
        eager = run(ni, nt, ng, scale=3.0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, eager)), seed


def test_two_graphs_do_not_share_a_workspace():
    graphs = []
    for seed, (tokens, vocab) in enumerate(((6000, 300), (900, 2000))):
        index, table, dy = make(tokens, vocab, 64, torch.float32, seed=seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(index, table, dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(index, table, dy)
        graphs.append((graph, out, (index, table, dy)))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for (graph, _, _), stream in zip(graphs, streams):    # both in flight
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, (index, table, dy) in graphs:
        assert all(torch.equal(a, e) for a, e in zip(out, run(index, table.detach().clone(), dy)))


def test_a_table_of_more_than_2_to_the_31_elements():
    """Offsets that pass 32 bits in the table, its gradient and the embedded tokens."""
    vocab, cols = 2**20 + 40000, 2048
    table = torch.zeros(vocab, cols, dtype=torch.float16, device=DEV)
    rows = torch.tensor([0, 5, 2**19, 2**20 - 1, 2**20, 2**20 + 1, vocab - 1], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    table[rows] = torch.randn(len(rows), cols, generator=g, device=DEV).half()
    index = rows[torch.randint(0, len(rows), (2**20 + 9000, ), generator=g, device=DEV)]
    dy = torch.zeros(len(index), cols, dtype=torch.float16, device=DEV)
    at = torch.tensor([0, 3, 2**20 - 1, 2**20, 2**20 + 1, len(index) - 1], device=DEV)
    dy[at] = torch.randn(len(at), cols, generator=g, device=DEV).half()
    table.requires_grad_()
    y = ea.embedding(index, table)
    assert torch.equal(y[at], table.detach()[index[at]]) and torch.equal(y[2**20 + 5], table.detach()[index[2**20 + 5]])
    d, = torch.autograd.grad(y, table, dy)
    want = torch.zeros(len(rows), cols, dtype=torch.float64, device=DEV)
    for i in at.tolist():
        want[(rows == index[i]).nonzero().item()] += dy[i].double()
    # at most six numbers that are not zero in a sum, so at most six roundings
    assert torch.all((d[rows].double() - want).abs() <= half_step(torch.float16, want) + 6 * 2.0**-24 * 6 * dy.abs().max().item())
    assert d.abs().sum(dtype=torch.float64).item() == d[rows].abs().sum(dtype=torch.float64).item()


def test_the_module_runs_the_kernel_and_falls_back(monkeypatch):
    from elixir_amd import fused_ops
    calls = []
    real = fused_ops.embedding
    monkeypatch.setattr(fused_ops, 'embedding', lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    torch.manual_seed(0)
    emb = ea.FusedEmbedding(30, 16, padding_idx=2, scale=4.0).to(DEV)
    index = torch.tensor([[1, 2, 29], [0, 2, 7]], device=DEV)
    assert torch.equal(emb(index), emb.weight[index] * 4) and calls == [1]
    emb(index).sum().backward()
    assert not emb.weight.grad[2].any() and (emb.weight.grad[29] == 4).all() and len(calls) == 2
    with torch.autocast('cuda', dtype=torch.float16):
        assert torch.equal(emb(index), emb.weight[index] * 4)
    emb.double()
    assert emb(index).dtype == torch.float64 and len(calls) == 2
    sparse = ea.FusedEmbedding(30, 16, sparse=True).to(DEV)
    sparse(index).sum().backward()
    assert sparse.weight.grad.is_sparse and len(calls) == 2


@pytest.mark.parametrize('tokens', [9000, 140000])
def test_large_vocabularies_and_many_tokens(tokens):
    """Three and four passes of the sort over several workgroups, up to the largest table; runs of one to many tokens."""
    for vocab, dtype in (((1 << 20) + 77, torch.float32), (1 << 30, torch.bfloat16)):
        g = torch.Generator(device=DEV).manual_seed(tokens)
        index = torch.randint(0, vocab, (tokens, ), generator=g, device=DEV)
        index[::3] = index[:5][torch.randint(0, 5, (len(index[::3]), ), generator=g, device=DEV)]
        index[7], index[8], index[9] = vocab - 1, 0, vocab - 1
        table = torch.zeros(vocab, 2, dtype=dtype, device=DEV)
        dy = torch.randn(tokens, 2, generator=g, device=DEV).to(dtype)
        d = run(index, table, dy)[1]
        named, inverse, count = torch.unique(index, return_inverse=True, return_counts=True)
        want = torch.zeros(len(named), 2, dtype=torch.float64, device=DEV).index_add_(0, inverse, dy.double())
        size = torch.zeros(len(named), 2, dtype=torch.float64, device=DEV).index_add_(0, inverse, dy.double().abs())
        tol = 2.0**-24 * (count[:, None] + 2) * size + half_step(dtype, want)
        assert torch.all((d[named].double() - want).abs() <= tol)
        d[named] = 0
        assert not d.any()


def test_hooks_that_hand_back_another_tensor_are_refused():
    index, table, dy = make(70, 40, 16, torch.float32)
    for unpack in (lambda t: t.int(), lambda t: t.cpu(), lambda t: t[:-1], lambda t: t.float()):
        table.requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = ea.embedding(index, table)
        with pytest.raises(RuntimeError, match='came back'):
            y.backward(dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack([t, t], 1)[:, 0]):    # another layout is fine
        y = ea.embedding(index, table)
    assert torch.equal(torch.autograd.grad(y, table, dy)[0], run(index, table.detach(), dy)[1])


def test_transforms_go_to_torch_or_are_refused():
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    index, table, _ = make(20, 30, 16, torch.float32)
    emb = ea.FusedEmbedding.from_pretrained(table, freeze=True)
    emb.scale = 2.0
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(table, torch.ones_like(table))
        with pytest.raises(NotImplementedError):
            ea.embedding(index, dual)
        assert torch.equal(emb(index), table[index] * 2)
    assert torch.equal(make_fx(lambda t: emb(t))(index)(index + 1), table[index + 1] * 2)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: ea.embedding(index, t).sum())(table)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('cols', [1, 5, 64, 96, 768, 770, 2048])
@pytest.mark.parametrize('tokens', [1, 2, 63, 64, 65, 257, 512, 1000, 1024, 1025, 2048, 2049])
def test_batches_around_the_changes_of_method(tokens, cols, dtype):
    """One launch without a sort, a sort by one workgroup, a sort by several: unique tokens, one token, two, and a padded half."""
    index, table, dy = make(tokens, 3000, cols, dtype, seed=tokens + cols, skew=1)
    index[:] = torch.randperm(3000, device=DEV)[:tokens]
    check(index, table, dy, scale=0.5)
    index[tokens // 2:] = 2999
    check(index, table, dy, padding_idx=2999)
    check(index, table, dy)
    index[:] = torch.arange(tokens, device=DEV) % 2
    check(index, table, dy)
    index[:] = -7    # outside: no gradient at all
    table.requires_grad_(False)
    assert not run(index, table, dy)[1].any()


@pytest.mark.parametrize('tokens, cols', [(7, 64), (1000, 64), (1000, 5), (1500, 64), (5000, 64)])
def test_graphs_of_every_method(tokens, cols):
    """Two graphs in flight on two streams, each replayed on new inputs, against eager passes."""
    graphs = []
    for seed in range(2):
        index, table, dy = make(tokens, 700, cols, torch.float16, seed=seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(index, table, dy, padding_idx=3)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(index, table, dy, padding_idx=3)
        graphs.append((graph, out, (index, table, dy)))
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(1, 4):
        new = [make(tokens, 700, cols, torch.float16, seed=10 * turn + i, skew=turn) for i in range(2)]
        for (_, _, static), fresh in zip(graphs, new):
            with torch.no_grad():
                for s, t in zip(static, fresh):
                    s.copy_(t)
        torch.cuda.synchronize()
        for (graph, _, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, out, _), fresh in zip(graphs, new):
            assert all(torch.equal(a, e) for a, e in zip(out, run(*fresh, padding_idx=3))), turn


def test_few_tokens_of_wide_and_long_tables():
    """One launch where offsets pass 32 bits, and at the largest table."""
    for vocab, cols, dtype in ((2**20 + 7, 4096, torch.bfloat16), (1 << 30, 4, torch.float16)):
        index = torch.tensor([vocab - 1, 0, 5, vocab - 1, vocab // 2, 5, vocab], device=DEV)
        dy = torch.randn(7, cols, device=DEV, dtype=torch.float32).to(dtype)
        table = torch.zeros(vocab, cols, dtype=dtype, device=DEV)
        d = run(index, table, dy)[1]
        want = {vocab - 1: dy[0].double() + dy[3].double(), 0: dy[1].double(), 5: dy[2].double() + dy[5].double(), vocab // 2: dy[4].double()}
        for row, value in want.items():
            assert torch.all((d[row].double() - value).abs() <= 4 * 2.0**-24 * dy.abs().max().item() * 2 + half_step(dtype, value))
            d[row] = 0
        assert not d.any()
        del d, table
