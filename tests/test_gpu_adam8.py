"""The Adam step over an 8-bit state on the GPU against the oracle (oracle/state8.py over the C oracle's fp32 step), at the
sizes and values where it can go wrong: identical bits in codes and exponents, master weights within ``near``."""
import numpy as np
import pytest
import torch

import elixir_amd as ea
from elixir_amd import _abi, _ops_abi
from elixir_amd import shapes as S
from elixir_amd.hybrid_adam import _read_state8, _write_state8, make_hyper_record
from helpers import CODE, from_bits, seeds, to_np
from oracle import oracle as O
from oracle import state8 as S8

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def bits(x: np.ndarray) -> np.ndarray:
    return x.view(np.uint32)


def same_f32(got, want, what):
    """Identical bits, any NaN like any other."""
    got, want = np.asarray(got, np.float32).ravel(), np.asarray(want, np.float32).ravel()
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), f'{what}: NaN pattern'
    assert np.array_equal(bits(got)[~nan], bits(want)[~nan]), f'{what}: {np.flatnonzero(bits(got) != bits(want))[:8]}'


def near(got, want, before, what):
    """Master weights after one step from the same ones (``before``).  The kernel takes the hardware's square root (1 ulp) and
    reciprocals (1 ulp each, of the denominator and of the bias correction), with three products or sums rounded to half an
    ulp beside them, the oracle rounds five times: relative to the change together less than 3 * 2^-23 + 8 * 2^-24 < 2^-20.
    On top each side rounds the weight once: 2 * 2^-24 of it.  Decay is part of ``want - before``, which only widens the
    first term.  Returns the kernel's weights, from which both sides go on."""
    got, want, before = (np.asarray(x, np.float32).ravel() for x in (got, want, before))
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), f'{what}: NaN pattern'
    g, w, b = (x[~nan].astype(np.float64) for x in (got, want, before))
    bad = np.abs(g - w) > 2.0**-20 * np.abs(w - b) + 2.0**-23 * np.abs(w)
    assert not bad.any(), f'{what}: {np.flatnonzero(bad)[:8]}, {np.abs(g - w).max()}'
    return got


def compare_codes(codes_m, codes_v, scales, want: S8.State8, what):
    """Codes (a NaN of exp_avg may carry either sign) and exponents."""
    m, v, e = to_np(codes_m).ravel(), to_np(codes_v).ravel(), to_np(scales)
    wm, wv = want.m.reshape(-1)[:want.n], want.v.reshape(-1)[:want.n]
    m = np.where((m & 0x7F) == 0x7F, 0x7F, m)
    for name, a, b in (('E of exp_avg', e[:, 0], want.me), ('E of exp_avg_sq', e[:, 1], want.ve), ('exp_avg', m, wm),
                       ('exp_avg_sq', v, wv)):
        assert np.array_equal(a.astype(np.int64), b.astype(np.int64)), f'{what} {name}: {np.flatnonzero(a != b)[:8]}'


@pytest.mark.parametrize('moment', [0, 1])
def test_read_and_write_against_the_definition(moment):
    """Every code under exponents from end to end; values over the whole fp32 range, subnormals, zeros, NaN and infinities."""
    every = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    e = np.arange(256)
    scales = np.stack([e, e], 1).astype(np.uint8)
    dm = torch.from_numpy(every).to(DEV)
    got = _read_state8(dm.view(-1), dm.view(-1), torch.from_numpy(scales).to(DEV), 0, every.size, torch.float32, torch.device('cuda', 0))
    with np.errstate(over='ignore'):
        want = S8.decode_sq(every, e) if moment else S8.decode_avg(every, e)
    same_f32(to_np(got[moment]), want, 'read')

    rng = np.random.default_rng(moment)
    x = (rng.standard_normal((300, 256)) * 10.0**rng.uniform(-44, 37, (300, 1)) * 10.0**rng.uniform(-12, 0, (300, 256))).astype(np.float32)
    x[0] = 0
    x[1, 5], x[2, 7], x[3, 9], x[4] = np.nan, np.inf, -np.inf, np.nan
    x[5, ::2] = 0
    x[6] = 2.0**-149
    x[7, 0] = 3.4e38
    if moment:
        x = np.abs(x)
    n = x.size - 101    # a partial block at the end
    flat = x.reshape(-1).copy()
    flat[n:] = 0
    x = flat.reshape(x.shape)
    codes = torch.full((x.size, ), 0xAB, dtype=torch.uint8, device=DEV)
    scales = torch.full((300, 2), 0xCD, dtype=torch.uint8, device=DEV)
    _write_state8(torch.from_numpy(flat).to(DEV), moment, codes[:n], scales, torch.device('cuda', 0))
    wc, we = S8.encode_sq(x, S8.HALF) if moment else S8.encode_avg(x)
    got = to_np(codes)
    assert np.all(got[n:] == 0xAB) and np.all(to_np(scales)[:, 1 - moment] == 0xCD)    # nothing else is touched
    assert np.array_equal(to_np(scales)[:, moment].astype(np.int64), we)
    got = got[:n] if moment else np.where((got[:n] & 0x7F) == 0x7F, 0x7F, got[:n])
    assert np.array_equal(got, wc.reshape(-1)[:n]), np.flatnonzero(got != wc.reshape(-1)[:n])[:8]


@pytest.mark.parametrize('begin,n', [(0, 1), (0, 256), (1, 1), (3, 7), (255, 2), (4, 1000), (250, 517), (1021, 3), (0, 4096), (512, 300)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_any_slice_is_read(begin, n, dtype):
    st = S8.State8(4096 + 77)
    rng = np.random.default_rng(n)
    st.set(rng.standard_normal(st.n).astype(np.float32), rng.random(st.n).astype(np.float32) * 1e-6)
    m, v = torch.from_numpy(st.m.reshape(-1)[:st.n].copy()).to(DEV), torch.from_numpy(st.v.reshape(-1)[:st.n].copy()).to(DEV)
    scales = torch.from_numpy(np.stack([st.me, st.ve], 1).astype(np.uint8)).to(DEV)
    got = _read_state8(m, v, scales, begin, begin + n, dtype, torch.device('cuda', 0))
    for t, want in zip(got, st.values()):
        assert t.dtype == dtype and t.numel() == n
        same_f32(to_np(t.float()), want[begin:begin + n], f'{begin} {n}')


SIZES = [1, 3, 255, 256, 257, 1000, 4096 + 13, 70001]


@pytest.mark.parametrize('adamw,wd,betas,bias', [(True, 0.0, (0.9, 0.999), True), (True, 0.1, (0.9, 0.95), True),
                                                 (False, 0.1, (0.4, 0.999), True), (True, 0.1, (0.9, 0.999), False)])
def test_standalone_steps_have_the_oracles_bits(oracle, adamw, wd, betas, bias):
    """Several tensors, one of them without a gradient, over steps of which the second and third repeat the first (the
    launch that rides its hyper records); div_scale none, a power of two and another number."""
    gen = torch.Generator().manual_seed(7)
    params = [torch.nn.Parameter((torch.randn(n, generator=gen) * 0.02).to(DEV)) for n in SIZES]
    idle = torch.nn.Parameter(torch.ones(5, device=DEV))
    opt = ea.HybridAdam(params[:3] + [idle] + params[3:], lr=1e-3, betas=betas, weight_decay=wd, adamw_mode=adamw,
                        bias_correction=bias, state_bits=8)
    pn = [to_np(p.data) for p in params]
    places = [0, 1, 2, 4, 5, 6, 7, 8]
    states = [S8.State8(n, salt) for n, salt in zip(SIZES, places)]
    for step, div in enumerate((-1, -1, 64.0, 48.0, -1), 1):
        scale = div if div > 0 else 1.0
        grads = [torch.randn(n, generator=gen) * 1e-2 * scale for n in SIZES]
        for p, g in zip(params, grads):
            if p.grad is None:
                p.grad = g.to(DEV)
            else:
                p.grad.copy_(g)
        opt.step(div_scale=div)
        for i, (p, g, st) in enumerate(zip(params, grads, states)):
            before = pn[i].copy()
            st.step(pn[i], g.numpy().copy(), O.F32, lr=1e-3, beta1=betas[0], beta2=betas[1], eps=1e-8, weight_decay=wd, step=step,
                    adamw_mode=adamw, bias_correction=bias, div_scale=div)
            got = opt.state[p]
            assert got['step'] == step
            pn[i] = near(to_np(p.data), pn[i], before, f'step {step} tensor {i} p')
            compare_codes(got['exp_avg'], got['exp_avg_sq'], got['scales'], st, f'step {step} tensor {i}')
            for t, want in zip(opt.read_moments(p), st.values()):
                assert t.shape == p.shape
                same_f32(to_np(t), want, f'step {step} tensor {i} values')
    assert torch.equal(idle.data, torch.ones(5, device=DEV)) and idle not in opt.state


@pytest.mark.parametrize('eps', [1e-8, 1e-12, 0.0])
def test_a_first_step_is_that_of_the_32_bit_state(eps):
    """From moments the codes hold (zeros) the master weights are those of the 32-bit state: within ``near``, and bit for bit
    where eps is so small that the kernel divides and takes roots exactly."""
    gen = torch.Generator().manual_seed(3)
    p0, g = torch.randn(10007, generator=gen) * 0.02, torch.randn(10007, generator=gen)
    g[:100] *= 1e-19
    out = []
    for state_bits in (8, 32):
        p = torch.nn.Parameter(p0.to(DEV))
        p.grad = g.to(DEV)
        ea.HybridAdam([p], lr=1e-3, weight_decay=0.1, eps=eps, state_bits=state_bits).step()
        out.append(to_np(p.data))
    near(out[0], out[1], p0.numpy(), 'first step')
    if eps < 2.0**-36:
        assert np.array_equal(bits(out[0]), bits(out[1]))


def test_gradients_that_are_not_finite(oracle):
    """inf and NaN spoil their own element, as in 32 bits, and no neighbour; what they leave stays NaN.  Very large and
    very small gradients, subnormal squares, a block of zeros."""
    n = 2048 + 100
    gen = torch.Generator().manual_seed(1)
    p = torch.nn.Parameter((torch.randn(n, generator=gen) * 0.02).to(DEV))
    opt = ea.HybridAdam([p], lr=1e-3, state_bits=8)
    pn, st = to_np(p.data), S8.State8(n)
    for step in range(1, 5):
        g = torch.randn(n, generator=gen) * 1e-2
        if step == 2:
            g[3], g[300], g[301], g[2147] = float('inf'), float('nan'), float('-inf'), float('nan')
        g[512:768] = 0
        g[768:1024] *= 1e-20
        g[1024:1280] *= 1e20
        g[1280] = 1e18
        p.grad = g.to(DEV)
        opt.step()
        before = pn.copy()
        st.step(pn, g.numpy().copy(), O.F32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0, step=step, adamw_mode=True)
        got = opt.state[p]
        pn = near(to_np(p.data), pn, before, f'step {step} p')
        compare_codes(got['exp_avg'], got['exp_avg_sq'], got['scales'], st, f'step {step}')
    m, v = opt.read_moments(p)
    assert torch.isnan(v).sum().item() == 4 and torch.isnan(m).sum().item() == 4


# ------------------------------------------------------------------------------------------------------------- chunk storage


def build8(named, chunk_size, dtype, *, seed=0, loss_scale=1.0, max_norm=0.0, weight_decay=0.0, lr=1e-3, host_resident=False,
           state_bits=8, **kw):
    sr = ea.greedy_search([(n, S.numel(s)) for n, s in named], chunk_size, dtype,
                          **(dict(shard_device=torch.device('cpu')) if host_resident else {}))
    if host_resident:
        for plan in sr.param_chunk_plans:
            plan.kwargs['cpu_pin_memory'] = True
    module = ea.ElixirModule(dict(named), sr, dtype=dtype)
    decay = [p for (n, s), p in zip(named, module.parameters()) if len(s) > 1]
    rest = [p for (n, s), p in zip(named, module.parameters()) if len(s) == 1]
    groups = [dict(params=g, weight_decay=w) for g, w in ((decay, weight_decay), (rest, 0.0)) if g]
    inner = ea.HybridAdam(groups, lr=lr, state_bits=state_bits)
    opt = ea.ElixirOptimizer(module, inner, initial_scale=loss_scale, hysteresis=1, max_norm=max_norm, **kw)
    gen = torch.Generator().manual_seed(seed)
    for pc in module.param_chunks:
        master = torch.zeros(pc.shard_size)
        master[:pc.utilized_size] = torch.randn(pc.utilized_size, generator=gen) * 0.02
        pc.paired_chunk.shard.copy_(master)
    return module, inner, opt, gen


def land(module, opt, gen, loss_scale, dtype, poison=None):
    """New gradients in every shard; returns them as numpy."""
    out = []
    for i, pc in enumerate(module.param_chunks):
        g = torch.zeros(pc.shard_size)
        g[:pc.utilized_size] = torch.randn(pc.utilized_size, generator=gen) * 1e-2 * loss_scale
        if poison is not None and i == 0:
            g[poison] = float('inf')
        g = g.to(dtype)
        pc.shard.copy_(g)
        pc.invalidate_stats()
        out.append(to_np(g))
    opt.mark_gradients_scaled()
    return out


def segments_of(opt, inner, chunk):
    out = []
    for group in inner.param_groups:
        for p in group['params']:
            if opt.param_to_optim_chunk[p] is chunk:
                out.append(opt.param_to_range[p] + (dict(weight_decay=group['weight_decay']), ))
    return sorted(out, key=lambda s: s[0])


NAMED = [('a', (130, 7)), ('b', (7, )), ('c', (3, )), ('d', (40, 41)), ('e', (1, )), ('f', (513, )), ('g', (257, 3)), ('h', (64, 64))]


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('graph', [False, True])
@pytest.mark.parametrize('chunk_size', [5000, 4099])
def test_chunked_steps_have_the_oracles_bits(oracle, dtype, graph, chunk_size):
    """Tensors that share blocks with their neighbours, two groups of hyper-parameters, padding at the end of a chunk;
    host-decided, device-decided and replayed from a recorded graph."""
    scale = 256.0 if dtype == torch.float16 else 1.0
    module, inner, opt, gen = build8(NAMED, chunk_size, dtype, loss_scale=scale, weight_decay=0.1)
    opt.graph_step = graph
    chunks = [pc.paired_chunk for pc in module.param_chunks]
    order = {c: i for i, c in enumerate(inner.binding.chunks)}
    pn = [to_np(c.shard) for c in chunks]
    st = [S8.State8(c.shard_size, order[c]) for c in chunks]
    for step in range(1, 7):
        opt.gated_step = graph or step % 2 == 0
        grads = land(module, opt, gen, scale, dtype)
        opt.step()
        assert opt.last_step_info['found_inf'] is False
        for i, (pc, c) in enumerate(zip(module.param_chunks, chunks)):
            before = pn[i].copy()
            st[i].step(pn[i], grads[i], CODE[dtype], segments_of(opt, inner, c), lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=step,
                       adamw_mode=True, div_scale=scale if scale != 1 else -1.0)
            m, v = inner.binding.moments(c)
            pn[i] = near(to_np(c.shard), pn[i], before, f'step {step} chunk {i} master')
            compare_codes(m, v, inner.binding.scales(c), st[i], f'step {step} chunk {i}')
            lowp = O.writeback(pn[i], CODE[dtype]) if dtype != torch.float32 else pn[i]
            assert np.array_equal(to_np(pc.shard).view(np.uint8), lowp.view(np.uint8)), f'step {step} chunk {i} writeback'


@pytest.mark.parametrize('gated', [True, False])
def test_a_skipped_step_leaves_the_state(gated):
    module, inner, opt, gen = build8(NAMED, 5000, torch.float16, loss_scale=256.0)
    opt.gated_step = gated
    land(module, opt, gen, 256.0, torch.float16)
    opt.step()
    before = [[t.clone() for t in (c.shard, *inner.binding.moments(c), inner.binding.scales(c))] for c in inner.binding.chunks]
    land(module, opt, gen, 256.0, torch.float16, poison=11)
    opt.step()
    assert opt.last_step_info['found_inf'] and opt.loss_scale == 128.0
    for c, kept in zip(inner.binding.chunks, before):
        for t, k in zip((c.shard, *inner.binding.moments(c), inner.binding.scales(c)), kept):
            assert torch.equal(t, k)
        assert torch.equal(c.paired_chunk.shard, c.shard.half())
    assert all(inner.state[p]['step'] == 1 for g in inner.param_groups for p in g['params'])
    # the step after a skipped one updates again (the armed table is disarmed)
    land(module, opt, gen, 128.0, torch.float16)
    opt.step()
    assert not torch.equal(inner.binding.chunks[0].shard, before[0][0])


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
def test_clipped_steps_follow_the_oracle(oracle, dtype):
    """With clipping the combined scale is a float64 sum in another order (1e-15 relative; the fp32 buffer of the norm can
    turn that into one fp32 unit, 2^-23): master weights are held to the change that unit can make in the step, at most
    2 * 2^-23 * |update| with |update| <= lr * (1 - beta1) / bc1 / (sqrt(1 - beta2) / sqrt(bc2)) = lr at the first step, on
    top of what ``near`` allows."""
    module, inner, opt, gen = build8(NAMED, 5000, dtype, loss_scale=64.0 if dtype == torch.float16 else 1.0, max_norm=0.05)
    lr = 1e-3
    scale = opt.loss_scale
    grads = land(module, opt, gen, scale, dtype)
    pn = [to_np(pc.paired_chunk.shard) for pc in module.param_chunks]
    opt.step()
    combined = opt.last_step_info['combined_scale']
    norm = np.sqrt(sum(O.sumsq(g, CODE[dtype]) for g in grads))
    assert combined == pytest.approx((norm / scale + 1e-6) / 0.05 * scale, rel=1e-6)
    for i, pc in enumerate(module.param_chunks):
        st = S8.State8(pc.shard_size, i)
        st.step(pn[i], grads[i], CODE[dtype], segments_of(opt, inner, pc.paired_chunk), lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=1,
                adamw_mode=True, div_scale=float(np.float32(combined)))
        got = to_np(pc.paired_chunk.shard)
        assert np.all(np.abs(got.astype(np.float64) - pn[i]) <= (2 * 2.0**-23 + 2.0**-20) * lr + np.abs(pn[i]) * 2.0**-23), i


def test_checkpoints_resume_with_the_same_bits_and_cross_the_two_widths():
    def run(module, opt, gen, steps):
        for _ in range(steps):
            land(module, opt, gen, 256.0, torch.float16)
            opt.step()

    module, inner, opt, gen = build8(NAMED, 5000, torch.float16, loss_scale=256.0, weight_decay=0.1)
    run(module, opt, gen, 3)
    saved = opt.state_dict()
    assert all(st['exp_avg'].dtype == torch.float32 and 'scales' not in st and st['step'] == 3 for st in saved['state'].values())
    masters = [c.shard.clone() for c in inner.binding.chunks]
    mark = gen.get_state()
    run(module, opt, gen, 3)

    again, inner2, opt2, gen2 = build8(NAMED, 5000, torch.float16, loss_scale=256.0, weight_decay=0.1, seed=9)
    run(again, opt2, gen2, 1)    # a state that the loaded one replaces
    opt2.load_state_dict(saved)
    for c, m in zip(inner2.binding.chunks, masters):
        c.shard.copy_(m)
    gen2.set_state(mark)
    for i, st in opt2.state_dict()['state'].items():
        assert torch.equal(st['exp_avg'], saved['state'][i]['exp_avg']) and torch.equal(st['exp_avg_sq'], saved['state'][i]['exp_avg_sq'])
    run(again, opt2, gen2, 3)
    for a, b in zip(inner.binding.chunks, inner2.binding.chunks):
        assert torch.equal(a.shard, b.shard)
        for x, y in zip(inner.binding.read_moments(a), inner2.binding.read_moments(b)):
            assert torch.equal(x, y)

    # the same checkpoint in a 32-bit optimizer: the values as they are; and from there into 8 bits again
    full, inner32, opt32, _ = build8(NAMED, 5000, torch.float16, loss_scale=256.0, state_bits=32)
    opt32.load_state_dict(saved)
    for i, st in opt32.state_dict()['state'].items():
        assert torch.equal(st['exp_avg'], saved['state'][i]['exp_avg'])
    c = inner32.binding.chunks[0]
    for t, flat in zip(inner32.binding.read_moments(c, torch.bfloat16), inner32.binding.moments(c)):
        assert torch.equal(t.float(), flat)
    fresh, inner4, opt4, _ = build8(NAMED, 4099, torch.float16, loss_scale=256.0)    # packed otherwise: other blocks
    opt4.load_state_dict(opt32.state_dict())
    for i, st in opt4.state_dict()['state'].items():
        want = saved['state'][i]['exp_avg']
        assert torch.all((st['exp_avg'] - want).abs() <= want.abs() * 2.0**-4 + want.abs().max() * 2.0**-10)


def test_standalone_state_dict_round_trip():
    gen = torch.Generator().manual_seed(2)
    params = [torch.nn.Parameter(torch.randn(n, generator=gen).to(DEV)) for n in (1000, 17)]
    opt = ea.HybridAdam(params, state_bits=8)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen).to(DEV)
    opt.step()
    opt.step()
    saved = opt.state_dict()
    twins = [torch.nn.Parameter(p.data.clone()) for p in params]
    twin = ea.HybridAdam(twins, state_bits=8)
    twin.load_state_dict(saved)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
        assert all(torch.equal(x, y) for x, y in zip(opt.read_moments(p), twin.read_moments(q)))
    opt.step()
    twin.step()
    assert all(torch.equal(p.data, q.data) for p, q in zip(params, twins))
    # a state put in place by hand has to be one the launches can address
    st = twin.state[twins[0]]
    twin.state[twins[0]] = dict(st, scales=st['scales'][:-1].clone())
    with pytest.raises(RuntimeError, match='scales'):
        twin.step()
    with pytest.raises(ValueError, match='elements'):
        ea.HybridAdam(twins, state_bits=8).load_state_dict(dict(saved, state={0: dict(saved['state'][1])}))


def test_shards_and_state_in_pinned_host_memory(oracle):
    module, inner, opt, gen = build8(NAMED, 5000, torch.float16, loss_scale=256.0, host_resident=True)
    pn = [to_np(pc.paired_chunk.shard) for pc in module.param_chunks]
    st = [S8.State8(pc.shard_size, i) for i, pc in enumerate(module.param_chunks)]
    for step in (1, 2):
        grads = land(module, opt, gen, 256.0, torch.float16)
        opt.step()
        torch.cuda.synchronize()
        for i, pc in enumerate(module.param_chunks):
            c = pc.paired_chunk
            assert all(t.is_pinned() for t in (*inner.binding.moments(c), inner.binding.scales(c)))
            before = pn[i].copy()
            st[i].step(pn[i], grads[i], O.F16, segments_of(opt, inner, c), lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=step,
                       adamw_mode=True, div_scale=256.0, weight_decay=0)
            pn[i] = near(to_np(c.shard), pn[i], before, f'step {step} chunk {i}')
            compare_codes(*inner.binding.moments(c), inner.binding.scales(c), st[i], f'step {step} chunk {i}')
    assert len(opt.state_dict()['state']) == len(NAMED)


def test_the_allocation_step_and_many_groups(oracle):
    """init_step: a step with zero gradients; 40 groups: hyper records through the table in device memory."""
    module, inner, opt, gen = build8(NAMED, 5000, torch.float32, init_step=True)
    assert all(inner.state[p]['step'] == 1 for g in inner.param_groups for p in g['params'])
    assert all(not t.any() for c in inner.binding.chunks for t in inner.binding.moments(c))
    params = [torch.nn.Parameter(torch.full((300, ), 0.5, device=DEV)) for _ in range(40)]
    opt = ea.HybridAdam([dict(params=[p], lr=1e-3 * (i + 1)) for i, p in enumerate(params)], state_bits=8)
    g = torch.randn(300, generator=gen)
    for p in params:
        p.grad = g.to(DEV)
    opt.step()
    for i, p in enumerate(params):
        pn, st = np.full(300, 0.5, np.float32), S8.State8(300, i)
        st.step(pn, g.numpy().copy(), O.F32, lr=1e-3 * (i + 1), beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0, step=1, adamw_mode=True)
        near(to_np(p.data), pn, np.full(300, 0.5, np.float32), f'group {i}')
        compare_codes(opt.state[p]['exp_avg'], opt.state[p]['exp_avg_sq'], opt.state[p]['scales'], st, f'group {i}')


@pytest.mark.parametrize('odd', [0, 1, 3])
def test_buffers_at_odd_offsets(oracle, odd):
    """The ABI on views that start at odd elements: the element-by-element path, same blocks and same bits."""
    n, dtype = 1500, torch.float16
    gen = torch.Generator().manual_seed(odd)
    hold = [torch.zeros(n + 8, dtype=t, device=DEV) for t in (dtype, dtype, torch.float32)]
    grad, low, master = (t[odd:odd + n] for t in hold)
    grad.copy_(torch.randn(n, generator=gen))
    master.copy_(torch.randn(n, generator=gen) * 0.02)
    m, v, scales = (torch.zeros(k, dtype=torch.uint8, device=DEV) for k in (n, n, 2 * 6))
    rows = np.zeros(1, _abi.CHUNK_DTYPE)
    segs = np.array([(0, 700, 0, 0), (800, n - 9, 0, 0)], dtype=_abi.SEG_DTYPE)
    rows[0] = (grad.data_ptr(), low.data_ptr(), master.data_ptr(), m.data_ptr(), v.data_ptr(), n, n - 5, 0, 0, 2)
    state = np.array([(scales.data_ptr(), 5, 9)], dtype=_ops_abi.STATE8_DTYPE)
    hyper = make_hyper_record(1e-3, 0.9, 0.999, 1e-8, 0.1, 4, True, True, 8)
    info = _abi.check_tables(rows, segs, 1, _abi.ELX_F16, _abi.ELX_F16)
    assert info.aligned == (odd == 0)
    _ops_abi.check_state8(rows, state)
    dev = [torch.from_numpy(t.view(np.uint8).copy()).to(DEV) for t in (rows, state, segs)]
    pn, gn = to_np(master), to_np(grad)
    before = pn.copy()
    _ops_abi.adam8_step_args_mt(dev[0].data_ptr(), dev[1].data_ptr(), 1, dev[2].data_ptr(), 2, hyper, info, -1.0, _abi.ELX_F16,
                                _abi.ELX_F16, 0, torch.cuda.current_stream().cuda_stream)
    st = S8.State8(n, 9)
    plain = S8.dither
    try:
        S8.dither = lambda blocks, salt, step: plain(np.asarray(blocks) + 5, salt, step)    # the row is blocks 5.. of its buffer
        st.step(pn, gn, O.F16, [(0, 700, {}), (800, n - 9, {})], lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, step=4,
                adamw_mode=True)
    finally:
        S8.dither = plain
    pn = near(to_np(master), pn, before, 'master')
    compare_codes(m, v, scales.view(-1, 2), st, f'odd {odd}')
    assert np.array_equal(to_np(low), O.writeback(pn, O.F16))
    for t, cut in zip(hold, (grad, low, master)):
        assert not t[:odd].any() and not t[odd + n:].any()


@pytest.mark.parametrize('seed', seeds(12))
def test_random_layouts(oracle, seed):
    rng = np.random.default_rng(seed)
    dtype = [torch.float16, torch.bfloat16, torch.float32][seed % 3]
    named = [(f't{i}', (int(rng.integers(1, 60)), int(rng.integers(1, 60))) if rng.random() < 0.7 else (int(rng.integers(1, 900)), ))
             for i in range(int(rng.integers(1, 12)))]
    chunk = max(S.numel(s) for _, s in named) + int(rng.integers(0, 4000))
    module, inner, opt, gen = build8(named, chunk, dtype, loss_scale=64.0, seed=seed, weight_decay=float(rng.choice([0, 0.1])))
    scale = opt.loss_scale
    pn = [to_np(pc.paired_chunk.shard) for pc in module.param_chunks]
    st = [S8.State8(pc.shard_size, i) for i, pc in enumerate(module.param_chunks)]
    for step in (1, 2):
        grads = land(module, opt, gen, scale, dtype)
        opt.step()
        for i, pc in enumerate(module.param_chunks):
            c = pc.paired_chunk
            before = pn[i].copy()
            st[i].step(pn[i], grads[i], CODE[dtype], segments_of(opt, inner, c), lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=step,
                       adamw_mode=True, div_scale=scale if scale != 1 else -1.0)
            pn[i] = near(to_np(c.shard), pn[i], before, f'step {step} chunk {i}')
            compare_codes(*inner.binding.moments(c), inner.binding.scales(c), st[i], f'step {step} chunk {i}')


def test_moments_follow_the_gradients_over_many_steps():
    """What the random rounding is for.  After 3000 steps on gradients of variance one, exp_avg_sq is an average of squares
    over the last thousand steps plus rounding noise: per step the chance of moving by one code (at most an eighth, on
    average a tenth of the value) is (1 - beta2) * 10 with sign, so the stationary standard deviation of one element is
    about sqrt(0.1 / 2) = 0.22 of the value, and the mean of 65536 independent elements has 0.22 / 256 < 0.001; the
    average of squares itself has 0.03 per element.  Held to 2 %.  Then the gradients stop: after 1000 more steps the mean
    has fallen to 0.999^1000 = 0.368 of what it was, within 3 %.  (Rounded to nearest, neither would have moved.)"""
    n = 65536
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = ea.HybridAdam([p], lr=1e-3, state_bits=8)
    p.grad = torch.empty(n, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(5)
    for _ in range(3000):
        p.grad.normal_(generator=gen)
        opt.step()
    v = opt.read_moments(p)[1]
    mean = v.mean().item()
    assert abs(mean / (1 - 0.999**3000) - 1) < 0.02, mean
    assert v.std().item() < 0.4
    p.grad.zero_()
    for _ in range(1000):
        opt.step()
    m, v = opt.read_moments(p)
    assert abs(v.mean().item() / mean / 0.999**1000 - 1) < 0.03, v.mean().item() / mean
    assert m.abs().max().item() < 1e-3


def test_a_buffer_of_more_than_2_to_the_32_elements(oracle):
    """One parameter whose offsets pass 32 bits.  Every 2^20 elements hold the same values, so master weights and the codes of
    exp_avg are those of one such stretch; exp_avg_sq is rounded by its place and is one of the two codes around its value.
    The last stretch, cut short, against the oracle."""
    stretch, n = 1 << 20, (1 << 32) + (1 << 20) + 77
    gen = torch.Generator().manual_seed(4)
    p0, g0 = torch.randn(stretch, generator=gen) * 0.02, torch.randn(stretch, generator=gen) * 1e-2
    reps = -(-n // stretch)
    p = torch.nn.Parameter(p0.to(DEV).repeat(reps)[:n].clone())
    p.grad = g0.to(DEV).repeat(reps)[:n].clone()
    opt = ea.HybridAdam([p], lr=1e-3, weight_decay=0.1, state_bits=8)
    opt.step()
    st = S8.State8(stretch, 0)
    pn = p0.numpy().copy()
    st.step(pn, g0.numpy().copy(), O.F32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, step=1, adamw_mode=True)
    first = p.data[:stretch]
    near(to_np(first), pn, p0.numpy(), 'first stretch')
    whole = p.data[:n - n % stretch].view(-1, stretch)
    assert torch.equal(whole, first.expand_as(whole)) and torch.equal(p.data[n - n % stretch:], first[:n % stretch])
    codes = opt.state[p]['exp_avg']
    assert np.array_equal(to_np(codes[:stretch]), st.m.reshape(-1))
    tail = n - n % stretch
    assert torch.equal(codes[(1 << 32):(1 << 32) + stretch], codes[:stretch])
    # the last block is cut short: its exponent may be another, so the values of its neighbours are compared
    assert torch.equal(codes[tail - 256:tail], codes[stretch - 256:stretch])
    m, v = opt.read_moments(p)
    assert torch.equal(m[(1 << 32) - 1000:(1 << 32) + 1000], m[:stretch].roll(1000)[:2000])
    v32 = np.float32(1.0 - 0.999) * g0.numpy() * g0.numpy()
    lo, hi = S8.decode_sq(*S8.encode_sq(S8.to_blocks(v32), np.zeros((stretch // 256, 256), np.int64))), \
        S8.decode_sq(*S8.encode_sq(S8.to_blocks(v32), np.full((stretch // 256, 256), (1 << 20) - 1, np.int64)))
    got = to_np(v[(1 << 32):(1 << 32) + stretch])
    slack = 2.0**-20    # the product above is rounded once less than the kernel's
    assert np.all(got >= lo.reshape(-1) * (1 - slack) - 1e-30) and np.all(got <= hi.reshape(-1) * (1 + slack) + 1e-30)
    block = (1 << 32) // 256 + 5    # and the dither of a block beyond 2^32 elements
    g = g0.numpy()[5 * 256:6 * 256]
    vv = np.zeros(256, np.float32)
    O.adam(g.copy(), O.F32, p0.numpy()[5 * 256:6 * 256].copy(), np.zeros(256, np.float32), vv, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
           weight_decay=0.1, step=1, adamw_mode=True)
    want, e = S8.encode_sq(vv[None], S8.dither(np.array([block]), 0, 1))
    assert np.array_equal(to_np(opt.state[p]['exp_avg_sq'][block * 256:(block + 1) * 256]), want[0])
    assert to_np(opt.state[p]['scales'])[block, 1] == e[0]
