"""The 8-bit optimizer state without a GPU: the code of the oracle against its definition, the tables and records of the
binding, and everything that is refused."""
import os
import re

import numpy as np
import pytest
import torch
from torch import nn

import elixir_amd as ea
from elixir_amd import _abi, _ops_abi
from elixir_amd.hybrid_adam import make_hyper_record
from elixir_amd.launch_plan import FlatBuffer, build_plan
from oracle import state8 as S8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_ops_library_exports_every_declared_symbol_and_carries_its_digest():
    text = re.sub(r'/\*.*?\*/', '', open(os.path.join(ROOT, 'include', 'elx_ops.h')).read(), flags=re.S)
    names = sorted(set(re.findall(r'\b(elx_[a-z0-9_]+)\s*\(', text)))
    lib = _ops_abi.load()
    assert sorted(_ops_abi.EXPORTS) == names
    for name in names:
        assert hasattr(lib, name)
    assert lib.elx_ops_source_sha().decode() == _ops_abi.source_sha16() == _ops_abi.built_source_sha(_ops_abi.LIB_PATH)


def test_a_stale_ops_library_is_refused(monkeypatch):
    from elixir_amd import build as B
    assert not B.is_stale()
    monkeypatch.setattr(_ops_abi, '_lib', None)
    monkeypatch.setattr(_ops_abi, 'source_sha16', lambda: '0123456789abcdef')
    with pytest.raises(RuntimeError, match='built from other sources'):
        _ops_abi.load()
    assert B.is_stale()


def _avg_value(code: int) -> float:
    """One byte of exp_avg from the definition of the format: sign, 4 exponent bits biased by 7, 3 mantissa bits."""
    sign, e, f = -1.0 if code & 0x80 else 1.0, (code >> 3) & 15, code & 7
    if e == 15 and f == 7:
        return float('nan')
    return sign * (f / 8 * 2.0**-6 if e == 0 else (1 + f / 8) * 2.0**(e - 7))


def _sq_value(code: int) -> float:
    e, f = code >> 3, code & 7
    if code == 255:
        return float('nan')
    return (f / 8 * 2.0**-126 if e == 0 else (1 + f / 8) * 2.0**(e - 127))


@pytest.mark.parametrize('e', [40, 100, 127, 190])
def test_every_code_stands_for_the_value_of_its_definition(e):
    codes = np.arange(256, dtype=np.uint8)[None]
    want = np.array([_avg_value(c) for c in range(256)]) * 2.0**(e - 135)
    np.testing.assert_array_equal(S8.decode_avg(codes, [e])[0].astype(np.float64), want)
    want = np.array([_sq_value(c) for c in range(256)]) * 2.0**(e - 31)
    np.testing.assert_array_equal(S8.decode_sq(codes, [e])[0].astype(np.float64), want)


def test_the_exponent_is_the_smallest_that_holds_the_largest_magnitude():
    for top, want in ((1.0, 127), (1.75, 127), (np.nextafter(np.float32(1.75), np.float32(2)), 128), (2.0, 128), (3.5, 128), (0.0, 0),
                      (1.5 * 2.0**-127, 0), (1.75 * 2.0**-127, 1), (1.0 * 2.0**-126, 1), (2.0**-149, 0), (3.0e38, 255)):
        x = np.zeros((1, 256), np.float32)
        x[0, 7] = -top
        assert S8.exponent(x)[0] == want, top
    x[0, :4] = (np.nan, np.inf, -np.inf, 0.5)
    x[0, 7] = 0
    assert S8.exponent(x)[0] == 126


def test_writing_what_was_read_changes_no_value():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((64, 256)) * 10.0**rng.uniform(-9, 3, (64, 256))).astype(np.float32)
    for encode, decode, data in ((S8.encode_avg, S8.decode_avg, x), (lambda t: S8.encode_sq(t, S8.HALF), S8.decode_sq, x * x)):
        once = decode(*encode(data))
        np.testing.assert_array_equal(decode(*encode(once)), once)
        # half a step of three mantissa bits, or the smallest quantum of the block: with the largest magnitude in
        # (0.875, 1.75] * 2^k that is 2^(k - 17) for exp_avg (14 binades of 8 codes below 2^k) and 2^(k - 33) for
        # exp_avg_sq, at most the largest / 0.875 * 2^-17 and * 2^-33; a whole one, because what is not zero stays above it
        floor = np.abs(data).max(1, keepdims=True) / 0.875 * (2.0**-17 if data is x else 2.0**-33)
        assert np.all(np.abs(once - data) <= np.maximum(np.abs(data) * 2.0**-4, floor))
        # bfloat16 holds every value
        t = torch.from_numpy(once.copy())
        assert torch.equal(t.to(torch.bfloat16).float(), t)


def test_random_rounding_has_the_right_expectation():
    """Over all 2^20 dithers a value between two codes is rounded up exactly as often as it should be; here over steps of
    the generator: 4096 steps x 256 elements, the mean within five standard deviations (a fraction q of the distance has
    standard deviation sqrt(q (1 - q) / N))."""
    q = 0.3
    x = np.full((1, 256), (1 + q / 8) * 0.5, np.float32)
    x[0, 0] = 1.0
    got = np.array([S8.decode_sq(*S8.encode_sq(x, S8.dither(np.array([3]), 1, step)))[0, 1:] for step in range(4096)])
    up = (got > 0.5).mean()
    assert set(np.unique(got)) == {np.float32(0.5), np.float32(0.5625)}
    assert abs(up - q) < 5 * np.sqrt(q * (1 - q) / got.size), up
    # and what is not zero stays above zero
    x[0, 1] = 2.0**-149
    assert np.all(S8.decode_sq(*S8.encode_sq(x, np.zeros((1, 256), np.int64)))[0, :2] > 0)


def test_hyper_records_carry_the_step_only_for_an_8_bit_state():
    args = (1e-3, 0.9, 0.999, 1e-8, 0.1, 70000, True, False)
    plain, eight = make_hyper_record(*args)[0], make_hyper_record(*args, 8)[0]
    assert plain['flags'] == _abi.ELX_HYPER_L2 and eight['flags'] == _abi.ELX_HYPER_L2 | 70000 << 8
    wrapped = make_hyper_record(1e-3, 0.9, 0.999, 1e-8, 0.0, (1 << 24) + 5, True, True, 8)[0]
    assert wrapped['flags'] == 5 << 8
    for name in plain.dtype.names:
        if name != 'flags':
            assert plain[name] == eight[name]


def test_the_plan_lists_one_state_row_per_update_row():
    base, tile = 1 << 40, _abi.tile_elems()
    n = 3 * 2048 * tile + 100
    bufs = [FlatBuffer(base, base, base + (1 << 32), base + (2 << 32), base + (3 << 32), n, n, [(0, n, 0)], scales=base + (4 << 32),
                       salt=i) for i in range(2)]
    plan = build_plan(bufs, 2, 2, 1, _abi.ELX_F16, _abi.ELX_F16)
    per = len(plan.rows) // 2
    assert len(plan.state_rows) == len(plan.rows) and per > 1
    for i, (row, st) in enumerate(zip(plan.rows, plan.state_rows)):
        at = (row['master'] - (base + (1 << 32))) // 4
        assert at % tile == 0
        assert row['m'] == base + (2 << 32) + at and row['v'] == base + (3 << 32) + at
        assert st['scales'] == base + (4 << 32) + 2 * (at // tile) and st['first_block'] == at // tile and st['salt'] == i // per
    bufs[1].scales = 0
    with pytest.raises(AssertionError):
        build_plan(bufs, 2, 2, 1, _abi.ELX_F16, _abi.ELX_F16)


def test_state_rows_are_checked():
    rows = np.zeros(1, _abi.CHUNK_DTYPE)
    rows[0] = (0, 0, 1 << 20, 1 << 21, 1 << 22, 1000, 1000, 0, 0, 0)
    good = np.array([(1 << 23, 0, 0)], dtype=_ops_abi.STATE8_DTYPE)
    _ops_abi.check_state8(rows, good)

    def expect(code, rows=rows, **edit):
        bad = good.copy()
        for k, val in edit.items():
            bad[k] = val
        with pytest.raises(_abi.ElxError) as e:
            _ops_abi.check_state8(rows, bad)
        assert e.value.code == code

    expect(_abi.ELX_E_NULL, scales=0)
    expect(_abi.ELX_E_ALIGN, scales=(1 << 23) + 1)
    expect(_abi.ELX_E_RANGE, first_block=(1 << 32) - 1)
    odd = rows.copy()
    odd['m'] += 2
    expect(_abi.ELX_E_ALIGN, rows=odd)


def test_launches_refuse_what_they_cannot_run():
    """Every refusal comes before anything is launched, so none of these needs a device."""
    L, at = _ops_abi.load(), 1 << 20
    info = _abi.TableInfo((4, 4, True))
    hyper = make_hyper_record(1e-3, 0.9, 0.999, 1e-8, 0.0, 1, True, True, 8)

    def refused(code, call, *args):
        with pytest.raises(_abi.ElxError) as e:
            call(*args)
        assert e.value.code == code

    F32, NONE = _abi.ELX_F32, _abi.ELX_NONE
    step = _ops_abi.adam8_step_mt
    refused(_abi.ELX_E_NULL, step, 0, at, 1, at, 1, at, 1, info, -1.0, F32, NONE, 0, 0)
    refused(_abi.ELX_E_NULL, step, at, 0, 1, at, 1, at, 1, info, -1.0, F32, NONE, 0, 0)
    refused(_abi.ELX_E_NULL, step, at, at, 1, at, 1, 0, 1, info, -1.0, F32, NONE, 0, 0)
    refused(_abi.ELX_E_SIZE, step, at, at, 0, at, 1, at, 1, info, -1.0, F32, NONE, 0, 0)
    refused(_abi.ELX_E_SIZE, step, at, at, 65536, at, 1, at, 1, info, -1.0, F32, NONE, 0, 0)
    refused(_abi.ELX_E_SIZE, step, at, at, 1, at, 1, at, 0, info, -1.0, F32, NONE, 0, 0)
    refused(_abi.ELX_E_TILES, step, at, at, 1, at, 1, at, 1, _abi.TableInfo((5, 4, True)), -1.0, F32, NONE, 0, 0)
    refused(_abi.ELX_E_DTYPE, step, at, at, 1, at, 1, at, 1, info, -1.0, 7, NONE, 0, 0)
    refused(_abi.ELX_E_DTYPE, step, at, at, 1, at, 1, at, 1, info, -1.0, _abi.ELX_F16, _abi.ELX_BF16, 0, 0)
    refused(_abi.ELX_E_SIZE, step, at, at, 1, at, 1, at, 1, info, -1.0, F32, NONE, 33, 0)
    assert L.elx_adam8_step_mt(at, at, 1, at, 1, at, 1, 4, 4, -1.0, F32, NONE, 64, 0, None) == _abi.ELX_E_RANGE
    refused(_abi.ELX_E_SIZE, _ops_abi.adam8_step_args_mt, at, at, 1, at, 1, np.concatenate([hyper] * 33), info, -1.0, F32, NONE, 0, 0)
    assert L.elx_adam8_step_args_mt(at, at, 1, at, 1, None, 1, 4, 4, -1.0, F32, NONE, 0, 0, None) == _abi.ELX_E_NULL
    refused(_abi.ELX_E_NULL, _ops_abi.adam8_step_gated_mt, at, 0, 1, at, 1, at, 1, info, F32, NONE, 0, 0)
    read, write = _ops_abi.state8_read, _ops_abi.state8_write
    refused(_abi.ELX_E_NULL, read, at, at, 0, 0, 4, at, at, F32, 0)
    refused(_abi.ELX_E_NULL, read, at, at, at, 0, 4, 0, 0, F32, 0)
    refused(_abi.ELX_E_NULL, read, 0, at, at, 0, 4, at, at, F32, 0)
    refused(_abi.ELX_E_DTYPE, read, at, at, at, 0, 4, at, at, _abi.ELX_F16, 0)
    refused(_abi.ELX_E_SIZE, read, at, at, at, 0, 0, at, at, F32, 0)
    refused(_abi.ELX_E_SIZE, read, at, at, at, 0, (1 << 33) + 1, at, at, F32, 0)
    refused(_abi.ELX_E_ALIGN, read, at, at, at, 0, 4, at + 2, at, F32, 0)
    refused(_abi.ELX_E_ALIGN, read, at + 1, at, at, 0, 4, at, at, F32, 0)
    refused(_abi.ELX_E_NULL, write, 0, 4, 0, at, at, 0)
    refused(_abi.ELX_E_RANGE, write, at, 4, 2, at, at, 0)
    refused(_abi.ELX_E_SIZE, write, at, 0, 0, at, at, 0)
    refused(_abi.ELX_E_ALIGN, write, at, 4, 0, at + 2, at, 0)


def test_the_optimizer_refuses_other_widths_and_cpu_parameters():
    p = nn.Parameter(torch.zeros(4))
    for bits in (16, 4, 0, None, '8'):
        with pytest.raises(ValueError, match='state_bits'):
            ea.HybridAdam([p], state_bits=bits)
    opt = ea.HybridAdam([p], state_bits=8)
    with pytest.raises(ValueError, match='no moments'):
        opt.read_moments(p)
    p.grad = torch.ones(4)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match='GPU'):
            opt.step()
    saved = dict(state={0: dict(step=3, exp_avg=torch.zeros(4), exp_avg_sq=torch.zeros(4))},
                 param_groups=ea.HybridAdam([p]).state_dict()['param_groups'])
    with pytest.raises(RuntimeError, match='GPU'):
        opt.load_state_dict(saved)
    with pytest.raises(TypeError, match='float16'):
        from elixir_amd.hybrid_adam import _as_read
        _as_read(p, p, torch.float16)
    assert ea.CPUAdam([p], state_bits=8).state_bits == 8 and ea.HybridAdam([p]).state_bits == 32


def test_bound_state_in_8_bits_without_a_gpu():
    """Chunk storage on the CPU: the layout of the state exists, reading or stepping it is refused."""
    net = nn.Linear(30, 20)
    sr = ea.greedy_search([(n, p.numel()) for n, p in net.named_parameters()], 700, torch.float16)
    module = ea.ElixirModule(net, sr, dtype=torch.float16)
    inner = ea.HybridAdam(net.parameters(), state_bits=8)
    opt = ea.ElixirOptimizer(module, inner)
    chunk = module.param_chunks[0].paired_chunk
    if chunk.shard.is_cuda:
        pytest.skip('a GPU is here: the GPU tests hold the values')
    m, v = inner.binding.moments(chunk)
    assert m.dtype == v.dtype == torch.uint8 and m.numel() == 700 and inner.binding.scales(chunk).shape == (3, 2)
    with pytest.raises(RuntimeError, match='GPU'):
        opt.state_dict()
    st = inner.state[inner.param_groups[0]['params'][1]]
    assert st['exp_avg'].numel() == 20 and st['scales'].shape == (1, 2)    # elements 600..619: block 2
    with pytest.raises(ValueError, match='elements'):
        inner.binding.read_moments(chunk, begin=5, end=701)
