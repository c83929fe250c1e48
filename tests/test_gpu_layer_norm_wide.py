"""layer_norm over many wide rows that are read element by element (odd widths, odd addresses): the backward kernels with 8 and 16
accesses per lane, which up to 1024 rows do not reach.  Reference and tolerances of test_gpu_layer_norm."""
import pytest
import torch

import elixir_amd as ea
from test_gpu_layer_norm import DEV, DTYPES, check, inputs, reference, run

pytestmark = pytest.mark.gpu


def verify(x, w, b, dy, got, dtype):
    for k, (want, tol) in reference(x, w, b, dy, 1e-5, dtype).items():
        if got[k] is not None:
            check(got[k], want, tol, k)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cols', [(1025, 513), (1025, 1025), (1030, 2049), (1025, 4095), (1025, 4097), (1300, 6001), (1025, 8191),
                                       (1025, 8193), (1026, 12289), (2000, 16383)])
def test_many_wide_rows_of_odd_widths(rows, cols, dtype):
    x, w, b, dy = inputs(rows, cols, dtype, seed=cols)
    got = dict(zip(('y', 'dx', 'dw', 'db'), run(x, w, b, dy)))
    verify(x, w, b, dy, got, dtype)
    again = dict(zip(('y', 'dx', 'dw', 'db'), run(x, w, b, dy)))
    assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('cols', [4096, 8192, 16384])
def test_many_wide_rows_at_odd_addresses(cols, dtype):
    """Even widths, but rows that start one element off: slices of wider tensors, read in place."""
    rows = 1025
    x, w, b, dy = inputs(rows, cols, dtype, seed=cols)
    wide_x, wide_dy = torch.zeros(rows, cols + 3, dtype=dtype, device=DEV), torch.zeros(rows, cols + 5, dtype=dtype, device=DEV)
    wide_x[:, 1:cols + 1], wide_dy[:, 3:cols + 3] = x, dy
    xs, dys = wide_x[:, 1:cols + 1].detach(), wide_dy[:, 3:cols + 3]
    got = dict(zip(('y', 'dx', 'dw', 'db'), run(xs, w, b, dys)))
    verify(x, w, b, dy, got, dtype)


@pytest.mark.parametrize('cols', [4097, 16383])
def test_some_gradients_of_wide_rows(cols):
    """Without dw and db there is no workspace and no second launch; without dx only they are written."""
    x, w, b, dy = inputs(1100, cols, torch.bfloat16, seed=5)
    full = run(x.clone(), w.clone(), b.clone(), dy)
    for wanted in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
        leaves = [t.detach().clone().requires_grad_(bool(k)) for t, k in zip((x, w, b), wanted)]
        got, = torch.autograd.grad(ea.layer_norm(*leaves), [t for t in leaves if t.requires_grad], dy)
        assert torch.equal(got, [f for f, k in zip(full[1:], wanted) if k][0])


@pytest.mark.parametrize('cols', [8193, 16383])
def test_rows_that_are_not_finite_stay_alone_in_wide_rows(cols):
    x, w, b, dy = inputs(1040, cols, torch.float32, seed=9)
    clean = run(x.clone(), w.clone(), b.clone(), dy)
    bad = x.detach().clone()
    bad[7, cols - 1], bad[1039, 0] = float('nan'), float('inf')
    y, dx, dw, db = run(bad, w.clone(), b.clone(), dy)
    others = [i for i in range(1040) if i not in (7, 1039)]
    assert torch.equal(y[others], clean[0][others]) and torch.equal(dx[others], clean[1][others]) and torch.equal(db, clean[3])
    assert torch.isnan(dx[[7, 1039]]).all() and torch.isnan(dw).all()
