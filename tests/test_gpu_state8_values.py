"""Values at the edges of the 8-bit state's code: each stays in its own element."""
import numpy as np
import pytest
import torch

import elixir_amd as ea
from elixir_amd.hybrid_adam import _read_state8, _write_state8
from helpers import to_np
from oracle import state8 as S8

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def write(x: np.ndarray, moment: int):
    """Codes and exponents of one moment as the library writes them."""
    codes = torch.zeros(x.size, dtype=torch.uint8, device=DEV)
    scales = torch.zeros(-(-x.size // S8.BLOCK), 2, dtype=torch.uint8, device=DEV)
    _write_state8(torch.from_numpy(x.reshape(-1).copy()).to(DEV), moment, codes, scales, torch.device('cuda', 0))
    return codes, scales


@pytest.mark.parametrize('bad', [-0.0, -1e-7, -3e-6, -1.0, -float('inf')])
@pytest.mark.parametrize('n', [256, 1024, 1000])
def test_a_sign_of_exp_avg_sq_stays_in_its_element(bad, n):
    """At every place of a lane's four elements, first and last of the block among them, and several side by side."""
    rng = np.random.default_rng(n)
    clean = (rng.random(n) * 1e-6 + 1e-8).astype(np.float32)
    for places in ([0], [1], [2], [3], [254], [255], [101, 102, 103, 104], [n - 1], range(0, n, 2)):
        x = clean.copy()
        x[list(places)] = bad
        codes, scales = write(x, 1)
        want, e = S8.encode_sq(S8.to_blocks(x), S8.HALF)
        assert np.array_equal(to_np(scales)[:, 1].astype(np.int64), e)
        assert np.array_equal(to_np(codes), want.reshape(-1)[:n]), (bad, places)
        # by themselves: the neighbours have the codes that the magnitude leaves them
        y = x.copy()
        if np.isfinite(bad):
            y[list(places)] = abs(bad)
            assert np.array_equal(to_np(codes), to_np(write(y, 1)[0]))


def test_a_checkpoint_with_such_values_spoils_no_neighbour():
    """Through load_state_dict, alone and bound to chunks: the other elements read as they do from a clean checkpoint."""
    n = 1000
    gen = torch.Generator().manual_seed(3)
    m, v = torch.randn(n, generator=gen) * 1e-3, torch.rand(n, generator=gen) * 1e-6 + 1e-8
    places = torch.tensor([0, 5, 255, 256, 514, 999])

    def alone():
        p = torch.nn.Parameter(torch.zeros(n, device=DEV))
        return ea.HybridAdam([p], state_bits=8), p

    def bound():
        module = ea.ElixirModule({'a': (n, )}, ea.greedy_search([('a', n)], 1100, torch.float16), dtype=torch.float16)
        inner = ea.HybridAdam(list(module.parameters()), state_bits=8)
        opt = ea.ElixirOptimizer(module, inner)
        return inner, (inner.param_groups[0]['params'][0], opt)

    for make in (alone, bound):
        got = []
        for bad in (0.0, -0.0):
            opt, p = make()
            sq = v.clone()
            sq[places] = bad
            opt.load_state_dict(dict(state={0: dict(step=3, exp_avg=m, exp_avg_sq=sq)}, param_groups=opt.state_dict()['param_groups']))
            got.append(opt.read_moments(p[0] if isinstance(p, tuple) else p))
        assert all(torch.equal(a, b) for a, b in zip(*got))
        assert not got[1][1][places].any()


LARGEST = float(np.finfo(np.float32).max)


@pytest.mark.parametrize('top', [LARGEST, 1.9375 * 2.0**127, 1.875 * 2.0**127, 1.75 * 2.0**127])
@pytest.mark.parametrize('moment', [0, 1])
def test_what_is_finite_stays_finite(top, moment):
    """Values next to the end of fp32, whose nearest code would stand for 2^128, between ordinary ones, an infinity and a NaN."""
    x = np.random.default_rng(1).random((3, 256)).astype(np.float32) * np.float32(1e38)
    x[0, [0, 77, 255]] = top
    x[1, 3], x[1, 4], x[1, 5] = top, np.inf, np.nan
    if moment == 0:
        x[:, 1::2] *= -1
    want, e = (S8.encode_sq(x, S8.HALF) if moment else S8.encode_avg(x))
    codes, scales = write(x, moment)
    got = to_np(codes).reshape(x.shape)
    got = got if moment else np.where((got & 0x7F) == 0x7F, 0x7F, got)
    assert np.array_equal(got, want) and np.array_equal(to_np(scales)[:, moment].astype(np.int64), e)
    values = _read_state8(codes, codes, scales, 0, x.size, torch.float32, torch.device('cuda', 0))[moment]
    finite = np.isfinite(x.reshape(-1))
    back = to_np(values)
    assert np.array_equal(np.isfinite(back), finite)
    # half a step of three mantissa bits; held at 1.875 * 2^127 the largest number of fp32 is off by a whole one
    assert np.all(np.abs(back[finite].astype(np.float64) / x.reshape(-1)[finite].astype(np.float64) - 1) <= 2.0**-4)
    again, scales2 = write(back, moment)
    assert torch.equal(again, codes) and torch.equal(scales2, scales)    # what was read is written back unchanged


def test_steps_with_squares_next_to_the_end_of_fp32():
    """exp_avg_sq of (1 - beta2) g^2 between 1.875 * 2^127 and the largest number: finite after every step, as in 32 bits."""
    n = 512
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = ea.HybridAdam([p], lr=1e-3, betas=(0.9, 0.999), state_bits=8)
    g = torch.full((n, ), 1e-3)
    g[::7] = 5.75e20    # 0.001 g^2 = 3.306e38
    g[3::7] = -5.7e20
    for step in range(1, 4):
        p.grad = (g if step == 1 else torch.full((n, ), 1e-3)).to(DEV)
        opt.step()
        m, v = opt.read_moments(p)
        assert torch.isfinite(m).all() and torch.isfinite(v).all() and torch.isfinite(p).all(), step
        assert v[::7].min() > 2.9e38 * 0.875
