"""layer_norm on the GPU, forward and backward, against the formulas in float64.

Tolerances, derived beforehand, in units u = 2^-24 (half a unit in the last place of fp32), with K = 72 additions at most on
the way of one element into a row sum (64 per lane or 16 per lane, 6 across lanes, 16 across wavefronts at most: 16 + 6 + 16 or
64 + 6 + ...), A = mean |x| of the row, h = (x - mean) rstd, t = dy w:
    mean            K u A
    h               dh = u (K A rstd + (K / 2 + 8) |h|): the mean's error, and half the relative error of the variance
    y               dh |w| + 4 u (|h w| + |b|), and the rounding to the tensor's type, half a step of it
    dx              rstd u (4 |t| + (K + 4) mean|t| + |h| (K + 4) mean|t h|) + rstd (|h| mean(|t| dh) + dh mean|t h|)
                    + (K / 2 + 8) u |dx|, and half a step
    dw, db          sum |dy| dh + R u sum |dy h| and R u sum |dy|, and half a step, where R = rows / 256 + 64 additions: a
                    lane's own rows (256 workgroups share them; fewer only where a workgroup then has at most 6), then 6 across
                    lanes, 16 row groups, 16 and 16 partial rows
An extra factor of 2 covers what is of second order in u."""
import pytest
import torch

import elixir_amd as ea

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U, K = 2.0**-24, 72
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dtype, ref):
    """Half a step of the type at ``ref``; in the subnormal range of fp16 the step is that of the smallest normal number."""
    return torch.finfo(dtype).eps / 2 * ref.abs().clamp_min(torch.finfo(dtype).tiny if dtype == torch.float16 else 0.0)


def reference(x, w, b, dy, eps, dtype):
    """(value, tolerance) of y, dx, dw, db in float64, on rows."""
    cols = x.shape[-1]
    rows = x.numel() // cols
    x, dy = x.detach().double().reshape(rows, cols), dy.detach().double().reshape(rows, cols)
    w = torch.ones(cols, dtype=torch.float64, device=x.device) if w is None else w.detach().double().reshape(-1)
    b = torch.zeros(cols, dtype=torch.float64, device=x.device) if b is None else b.detach().double().reshape(-1)
    mean = x.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    h = (x - mean) * rstd
    A = x.abs().mean(1, keepdim=True)
    dh = U * (K * A * rstd + (K / 2 + 8) * h.abs())
    y = h * w + b
    t = dy * w
    mt, mth = t.mean(1, keepdim=True), (t * h).mean(1, keepdim=True)
    at, ath = t.abs().mean(1, keepdim=True), (t * h).abs().mean(1, keepdim=True)
    dx = rstd * (t - mt - h * mth)
    ddx = (rstd * U * (4 * t.abs() + (K + 4) * at + h.abs() * (K + 4) * ath) + rstd * (h.abs() * (t.abs() * dh).mean(1, keepdim=True) + dh * ath)
           + (K / 2 + 8) * U * dx.abs())
    R = rows / 256 + 64
    dw, db = (dy * h).sum(0), dy.sum(0)
    out = dict(y=(y, dh * w.abs() + 4 * U * ((h * w).abs() + b.abs())), dx=(dx, ddx),
               dw=(dw, (dy.abs() * dh).sum(0) + R * U * (dy * h).abs().sum(0)), db=(db, R * U * dy.abs().sum(0)))
    return {k: (v, 2 * tol + half_step(dtype, v)) for k, (v, tol) in out.items()}


def check(got, want, tol, what):
    got = got.detach().double().reshape(want.shape)
    big = want.abs() > 65504 if want.dtype == torch.float64 else None
    bad = (got - want).abs() > tol
    bad |= ~torch.isfinite(got) & ~(big if big is not None else False)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {got.numel()}, worst {(got - want).abs().max().item():.3g}'


def run(x, w, b, dy, eps=1e-5):
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_()
    y = ea.layer_norm(x, w, b, eps)
    grads = list(torch.autograd.grad(y, leaves, dy))
    return y, grads.pop(0), grads.pop(0) if w is not None else None, grads.pop(0) if b is not None else None


def inputs(rows, cols, dtype, seed=0, offset=1.0, shape=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)    # noqa: E731
    x = rnd(rows, cols) * (0.2 + 3 * torch.rand(rows, 1, generator=g, device=DEV)) + offset * rnd(rows, 1)
    return x.to(dtype), (1 + 0.2 * rnd(cols)).to(dtype), (0.2 * rnd(cols)).to(dtype), (rnd(rows, cols) * 0.1).to(dtype)


COLS = [1, 2, 7, 8, 16, 63, 64, 65, 256, 257, 512, 520, 768, 769, 1000, 1024, 1032, 2048, 2052, 4096, 4097, 5000, 8192, 11008, 16383, 16384]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('cols', COLS)
@pytest.mark.parametrize('rows', [1, 5, 37])
def test_every_width(rows, cols, dtype):
    x, w, b, dy = inputs(rows, cols, dtype, seed=cols)
    got = dict(zip(('y', 'dx', 'dw', 'db'), run(x, w, b, dy)))
    for k, (want, tol) in reference(x, w, b, dy, 1e-5, dtype).items():
        check(got[k], want, tol, k)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cols', [(2047, 769), (4096, 64), (1023, 2048), (1025, 4096), (20000, 24), (8192, 1024), (5000, 1000),
                                       (70001, 128), (30000, 8), (30001, 17), (700, 11008)])
def test_many_rows(rows, cols, dtype):
    x, w, b, dy = inputs(rows, cols, dtype, seed=rows)
    got = dict(zip(('y', 'dx', 'dw', 'db'), run(x, w, b, dy)))
    for k, (want, tol) in reference(x, w, b, dy, 1e-5, dtype).items():
        check(got[k], want, tol, k)
    again = dict(zip(('y', 'dx', 'dw', 'db'), run(x, w, b, dy)))
    assert all(torch.equal(got[k], again[k]) for k in got)    # the order of every sum is fixed


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('with_w,with_b', [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(with_w, with_b, dtype):
    x, w, b, dy = inputs(300, 768, dtype)
    w, b = w if with_w else None, b if with_b else None
    got = dict(zip(('y', 'dx', 'dw', 'db'), run(x, w, b, dy)))
    for k, (want, tol) in reference(x, w, b, dy, 1e-5, dtype).items():
        if got[k] is not None:
            check(got[k], want, tol, k)
    assert (got['dw'] is None) == (not with_w) and (got['db'] is None) == (not with_b)


def test_only_some_gradients_are_wanted():
    x, w, b, dy = inputs(100, 512, torch.float32)
    full = run(x.clone(), w.clone(), b.clone(), dy)
    for wanted in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)):
        leaves = [t.detach().clone().requires_grad_(bool(k)) for t, k in zip((x, w, b), wanted)]
        y = ea.layer_norm(*leaves)
        got = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)
        assert all(torch.equal(g, f) for g, f in zip(got, [f for f, k in zip(full[1:], wanted) if k]))
    with torch.no_grad():
        assert torch.equal(ea.layer_norm(x, w, b), full[0]) and not ea.layer_norm(x, w, b).requires_grad


@pytest.mark.parametrize('dtype', DTYPES)
def test_a_large_mean_costs_no_digits_but_its_own(dtype):
    """Rows around 1000 with a spread of one, constant rows, rows of zeros, tiny rows against eps."""
    x, w, b, dy = inputs(64, 1024, dtype, offset=0.0)
    x = x.float()
    x[:16] += 1000.0
    x[16:24] = 3.0
    x[24:32] = 0.0
    x[32:40] *= 1e-4
    x = x.to(dtype)
    got = dict(zip(('y', 'dx', 'dw', 'db'), run(x, w, b, dy)))
    for k, (want, tol) in reference(x, w, b, dy, 1e-5, dtype).items():
        check(got[k], want, tol, k)


def test_rows_that_are_not_finite_stay_alone():
    x, w, b, dy = inputs(8, 300, torch.float32)
    x[2, 7], x[5, 0] = float('nan'), float('inf')
    y = ea.layer_norm(x, w, b)
    clean = x.clone()
    clean[2], clean[5] = 1.0, 1.0
    want = ea.layer_norm(clean, w, b)
    keep = [0, 1, 3, 4, 6, 7]
    assert torch.equal(y[keep], want[keep]) and torch.isnan(y[2]).all() and torch.isnan(y[5]).all()


@pytest.mark.parametrize('dtype', DTYPES)
def test_strides_shapes_and_alignment(dtype):
    """Slices read in place, inputs that have to be copied, gradients that arrive expanded, odd offsets, several trailing
    dimensions, leading dimensions of one or none."""
    base, w, b, dy = inputs(60, 1040, dtype)
    for x in (base[:, :1024], base[:, 3:1027], base[::3, 16:], base.view(6, 10, 1040)[:, ::2, 8:], base.t()[:50], base[4], base[:1, :7],
              base.view(3, 4, 5, 1040)[1:, :, :, 16:]):
        cols = x.shape[-1]
        x = x.detach()
        ww, bb = w.detach()[:cols].clone(), b.detach()[:cols].clone()
        g = torch.randn(x.shape, device=DEV).to(dtype)
        got = dict(zip(('y', 'dx', 'dw', 'db'), run(x, ww, bb, g)))
        assert got['y'].shape == x.shape and got['y'].is_contiguous()
        for k, (want, tol) in reference(x, ww, bb, g, 1e-5, dtype).items():
            check(got[k], want, tol, f'{tuple(x.shape)} {x.stride()} {k}')
    x = base[:, :1024].detach()
    wide = torch.ones(1, dtype=dtype, device=DEV).expand(60, 1024)    # sum().backward()
    ww, bb = w.detach()[:1024].clone(), b.detach()[:1024].clone()
    got = dict(zip(('y', 'dx', 'dw', 'db'), run(x, ww, bb, wide)))
    for k, (want, tol) in reference(x, ww, bb, wide, 1e-5, dtype).items():
        check(got[k], want, tol, 'expanded ' + k)
    odd = torch.zeros(1025, dtype=dtype, device=DEV)[1:]    # weight and bias at an odd address
    odd.copy_(w.detach()[:1024])
    check(ea.layer_norm(x, odd, bb), *reference(x, ww, bb, wide, 1e-5, dtype)['y'], 'odd weight')    # another order of the sums
    two = base[:, :1024].detach().reshape(60, 32, 32)
    w2, b2 = ww.view(32, 32), bb.view(32, 32)
    assert torch.equal(ea.layer_norm(two, w2, b2).reshape(60, 1024), ea.layer_norm(two.reshape(60, 1024), ww, bb))
    assert torch.equal(ea.layer_norm(two, normalized_shape=(32, 32)), ea.layer_norm(two.reshape(60, 1024)).view(60, 32, 32))


def test_empty_batches():
    x = torch.zeros(0, 5, 64, device=DEV, requires_grad=True)
    w, b = torch.ones(64, device=DEV, requires_grad=True), torch.zeros(64, device=DEV, requires_grad=True)
    y = ea.layer_norm(x, w, b)
    assert y.shape == (0, 5, 64)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert dx.shape == x.shape and not dw.any() and not db.any() and dw.shape == w.shape


def test_refusals_on_device_tensors():
    x, w, b, _ = inputs(4, 64, torch.float32)
    with pytest.raises(TypeError, match='float64'):
        ea.layer_norm(x.double())
    with pytest.raises(TypeError, match='float16'):
        ea.layer_norm(x, w.half(), b.half())
    with pytest.raises(RuntimeError, match='GPU'):
        ea.layer_norm(x, w.cpu(), b)
    with pytest.raises(ValueError, match='16384'):
        ea.layer_norm(torch.zeros(1, 16385, device=DEV))
    with pytest.raises(ValueError, match='elements'):
        ea.layer_norm(torch.zeros(4, 0, device=DEV))


def test_a_gradient_can_be_differentiated():
    """A penalty on the gradient: through torch's operators, so the second derivatives are torch's."""
    out = []
    for f in (lambda x, w, b: ea.layer_norm(x, w, b), lambda x, w, b: torch.nn.functional.layer_norm(x, (64, ), w, b)):
        x, w, b, c = (t.detach() for t in inputs(6, 64, torch.float32))
        leaves = [t.requires_grad_() for t in (x, w, b)]
        g = torch.autograd.grad((f(*leaves) * c).square().sum(), leaves, create_graph=True)
        out.append([*g, *torch.autograd.grad(sum(t.square().sum() for t in g), leaves)])
    for got, want in zip(*out):
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4 * want.abs().max().item())


def test_gradients_against_differences():
    """Directional derivatives of sum(c y): the kernel's gradient against central differences of the kernel's forward.  The
    differences are off by what those of float64 are off (measured on the float64 formula) and by the rounding of the two
    outputs, at most sum |c| tol_y each, over the step 2 s."""
    x, w, b, c = (t.detach() for t in inputs(7, 193, torch.float32, seed=3))
    y, dx, dw, db = run(x.clone(), w.clone(), b.clone(), c)
    ref = reference(x, w, b, c, 1e-5, torch.float32)
    g = torch.Generator(device=DEV).manual_seed(11)
    s = 2.0**-7
    forward64 = lambda x, w, b: reference(x, w, b, c, 1e-5, torch.float32)['y'][0].reshape(x.shape)    # noqa: E731
    for i, grad in enumerate((dx, dw, db)):
        args = [x, w, b]
        d = torch.randn(args[i].shape, generator=g, device=DEV).mul(8).round().div(8)    # few bits: x + s d is nearly exact
        plus, minus = list(args), list(args)
        plus[i], minus[i] = args[i] + s * d, args[i] - s * d
        step = (plus[i].double() - minus[i].double())    # what the two really differ by
        slope = ((ea.layer_norm(*plus).double() - ea.layer_norm(*minus).double()) * c.double()).sum()
        slope64 = ((forward64(*plus) - forward64(*minus)) * c.double()).sum()
        truncation = (slope64 - (ref[('dx', 'dw', 'db')[i]][0].reshape(step.shape) * step).sum()).abs()
        noise = 2 * (c.double().abs().reshape(7, 193) * ref['y'][1]).sum() * 2
        tol_grad = (ref[('dx', 'dw', 'db')[i]][1].reshape(step.shape) * step.abs()).sum()
        assert (slope - (grad.double() * step).sum()).abs() <= truncation + noise + tol_grad
        assert noise < 0.05 * (grad.double().abs() * step.abs()).sum()    # the test says something


def test_streams_and_graphs():
    """On a side stream; several calls in flight on two streams; forward and backward captured and replayed on new inputs,
    with eager work between the replays."""
    x, w, b, dy = (t.detach() for t in inputs(513, 768, torch.bfloat16))
    want = run(x.clone(), w.clone(), b.clone(), dy)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            results.append(run(x.clone(), w.clone(), b.clone(), dy))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, e) for a, e in zip(r, want))
    sx, sw, sb, sg = (t.clone() for t in (x, w, b, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(sx, sw, sb, sg)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(sx, sw, sb, sg)
    for seed in range(1, 5):
        nx, nw, nb, ng = (t.detach() for t in inputs(513, 768, torch.bfloat16, seed=seed))
        with torch.no_grad():
            for s, t in zip((sx, sw, sb, sg), (nx, nw, nb, ng)):
                s.copy_(t)
        graph.replay()
        eager = run(nx, nw, nb, ng)
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, eager)), seed


def test_two_graphs_do_not_share_a_workspace():
    graphs = []
    for seed, (rows, cols) in enumerate(((700, 512), (300, 2048))):
        args = [t.detach() for t in inputs(rows, cols, torch.float32, seed=seed)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(*args)
        graphs.append((graph, out, args))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for (graph, _, _), stream in zip(graphs, streams):    # both in flight
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, args in graphs:
        assert all(torch.equal(a, e) for a, e in zip(out, run(*[t.detach().clone() for t in args])))


def test_saved_tensor_hooks_checkpointing_and_anomaly_mode():
    """What calls back into Python from inside the extension."""
    x, w, b, dy = inputs(40, 96, torch.float32)
    want = run(x.clone(), w.clone(), b.clone(), dy)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    with torch.autograd.graph.save_on_cpu():
        y = ea.layer_norm(*leaves)
    assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(y, leaves, dy), want[1:]))
    y = torch.utils.checkpoint.checkpoint(ea.layer_norm, *leaves, use_reentrant=False)
    assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(y, leaves, dy), want[1:]))
    with torch.autograd.set_detect_anomaly(True):
        assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(ea.layer_norm(*leaves), leaves, dy), want[1:]))
    with torch.inference_mode():
        assert torch.equal(ea.layer_norm(x, w, b), want[0])


def test_more_than_2_to_the_32_elements():
    """Rows whose offsets pass 32 bits, in elements and in bytes; the last and some in between against float64."""
    rows, cols = 2**31 // 1024 + 2**31 // 1024 + 3, 1024
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    pick = torch.tensor([0, 1, 2**21 - 1, 2**21, 2**21 + 1, 2**22 - 1, 2**22, rows - 1], device=DEV)
    x.zero_()
    x[pick] = torch.randn(len(pick), cols, generator=g, device=DEV).bfloat16()
    w, b = (1 + 0.1 * torch.randn(cols, generator=g, device=DEV)).bfloat16(), torch.randn(cols, generator=g, device=DEV).bfloat16()
    dy = torch.zeros_like(x)
    dy[pick] = torch.randn(len(pick), cols, generator=g, device=DEV).bfloat16()
    y, dx, dw, db = run(x, w, b, dy)
    ref = reference(x[pick], w, b, dy[pick], 1e-5, torch.bfloat16)
    check(y[pick], *ref['y'], 'y')
    check(dx[pick], *ref['dx'], 'dx')
    check(dw, *ref['dw'], 'dw')    # rows of zeros add nothing
    check(db, *ref['db'], 'db')
    assert torch.equal(y[5], b) and torch.equal(y[2**22 + 1], b) and not dx[2**22 + 1].any()


def test_the_module_runs_the_kernel_and_falls_back(monkeypatch):
    from elixir_amd import fused_ops
    calls = []
    real = fused_ops.layer_norm
    monkeypatch.setattr(fused_ops, 'layer_norm', lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    torch.manual_seed(0)
    norm = ea.FusedLayerNorm(48).to(DEV)
    plain = torch.nn.LayerNorm(48).to(DEV)
    x = torch.randn(5, 48, device=DEV)
    torch.testing.assert_close(norm(x), plain(x), rtol=1e-5, atol=1e-5)
    assert calls == [1]
    with torch.autocast('cuda', dtype=torch.float16):
        assert torch.equal(norm(x), plain(x))
    assert torch.equal(norm.double()(x.double()), plain.double()(x.double()))
    norm, plain = norm.float(), plain.float()
    assert torch.equal(torch.func.vmap(norm)(x), torch.func.vmap(plain)(x))
    with pytest.raises(RuntimeError):
        norm(x[:, :40])
    assert calls == [1]


def test_hooks_that_hand_back_another_tensor_are_refused():
    """The backward launch reads what the hooks of the saved tensors return: another type, size or device is an error."""
    def loss(unpack):
        leaves = [t.requires_grad_() for t in inputs(40, 96, torch.float32)[:3]]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            return ea.layer_norm(*leaves).sum()

    for unpack in (lambda t: t.half(), lambda t: t.cpu(), lambda t: t[:1].clone(), lambda t: t.t() if t.dim() == 2 and len(t) == 40 else t):
        with pytest.raises(RuntimeError, match='came back'):
            loss(unpack).backward()
    loss(lambda t: t.t().contiguous().t() if t.dim() == 2 else t).backward()    # another layout is fine


def test_negated_views():
    """A view that negates what lies in memory (the imaginary part of a conjugate) is read as what it stands for."""
    z = torch.randn(6, 1, 33, dtype=torch.complex64, device=DEV).conj()
    x = z.imag.transpose(0, 1)[0]
    assert x.is_neg()
    w = torch.randn(33, device=DEV)
    lazy = torch._neg_view(x.neg().contiguous())
    for t in (x, lazy):
        want = ea.layer_norm(x.clone().contiguous().resolve_neg(), w)
        assert torch.equal(ea.layer_norm(t, w), want)
    assert torch.equal(ea.layer_norm(x.resolve_neg(), torch._neg_view(w.neg())), ea.layer_norm(x.resolve_neg(), w))


def test_transforms_go_to_torch_or_are_refused():
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, b, _ = (t.detach() for t in inputs(5, 48, torch.float32))
    norm = ea.FusedLayerNorm(48).to(DEV).requires_grad_(False)
    plain = torch.nn.LayerNorm(48).to(DEV).requires_grad_(False)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, b.expand(5, 48).contiguous())
        got, want = forward_ad.unpack_dual(norm(dual)), forward_ad.unpack_dual(plain(dual))
        assert torch.equal(got.tangent, want.tangent) and torch.equal(got.primal, want.primal)
        with pytest.raises(NotImplementedError):
            ea.layer_norm(dual, w, b)
    for traced in (make_fx(lambda t: norm(t))(x), torch.jit.trace(norm, x, check_trace=False)):
        other = torch.randn(5, 48, device=DEV)
        assert torch.equal(traced(other), plain(other))
    for call in (lambda: torch.func.vmap(lambda t: ea.layer_norm(t, w, b))(x.view(5, 1, 48)),
                 lambda: torch.func.grad(lambda t: ea.layer_norm(x, t, b).sum())(w)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', [2, 15, 17, 255, 1023, 1024, 1025])
@pytest.mark.parametrize('cols', [8, 64, 769, 2049, 3080, 11008])
def test_rows_around_the_change_of_method(rows, cols, dtype):
    """One launch for dx and the sums, or two; strided rows; each gradient alone."""
    x, w, b, dy = inputs(rows, cols, dtype, seed=rows + cols)
    wide = torch.zeros(rows, cols + 8, dtype=dtype, device=DEV)
    wide[:, :cols] = x
    x = wide[:, :cols].detach()
    got = run(x, w, b, dy)
    ref = reference(x, w, b, dy, 1e-5, dtype)
    for name, t in zip(('y', 'dx', 'dw', 'db'), got):
        check(t, *ref[name], name)
    y = ea.layer_norm(x, w, b)
    for i, leaf in enumerate((x, w, b)):
        assert torch.equal(torch.autograd.grad(y, leaf, dy, retain_graph=True)[0], got[1 + i])


@pytest.mark.parametrize('rows, cols', [(1, 2048), (1024, 96), (1025, 96), (3000, 2048)])
def test_graphs_of_both_methods(rows, cols):
    """Two graphs in flight on two streams, each replayed on new inputs, against eager passes."""
    graphs = []
    for seed in range(2):
        static = [t.detach() for t in inputs(rows, cols, torch.float16, seed=seed)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(*static)
        graphs.append((graph, out, static))
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(1, 4):
        new = [[t.detach() for t in inputs(rows, cols, torch.float16, seed=10 * turn + i)] for i in range(2)]
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
            assert all(torch.equal(a, e) for a, e in zip(out, run(*fresh))), turn
