"""Cases, plain forms and 64-bit forms of the operators of a training step beside the optimizer step in 32 bits:

  adam8       the AdamW step whose exp_avg and exp_avg_sq are held in 8 bits, over many tensors (``HybridAdam(state_bits=8)``)
              or over chunk storage (``ElixirOptimizer``: landing, overflow flags, clipping, update, low-precision copy)
  layer_norm  layer norm, forward and backward, with the reduction of the gradients of weight and bias
  embedding   embedding lookup with scaling, and the dense gradient of its table

``own`` chooses between the plain form (elementary torch operations, in 32 bits) and the framework's operators.

The 8-bit state.  A buffer is cut into blocks of 256 elements.  A block of exp_avg holds one exponent byte E and 256 codes in
the format torch calls float8_e4m3fn, standing for  code * 2^(E - 135);  a block of exp_avg_sq holds one exponent byte and 256
unsigned codes of 5 exponent and 3 mantissa bits, standing for  float32(bits = code << 20) * 2^(E - 31).  E is the smallest
exponent for which the largest magnitude of the block is at most 1.75 * 2^(E - 127).  exp_avg is rounded to nearest even.
exp_avg_sq moves by a thousandth of itself in a step, far less than the distance of two codes, and is rounded at random with
the right expectation: up or down by the 20 bits that ``_dither`` gives for (buffer, block, element, step); what is not zero
stays above zero.  Every value of either code is a bfloat16 number too, and that is how the state is returned.
"""
import math

import torch

own = False

BLOCK = 256
DTYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
ESIZE = {'float32': 4, 'float16': 2, 'bfloat16': 2}
LR, BETAS, EPS, DECAY = 5e-5, (0.9, 0.999), 1e-8, 0.01
FIRST_STEP = 500    # the moments are those of a run under way


# ---------------------------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # biases and norm weights of odd lengths, fine-tuned on their own: nothing but latency
        dict(name='adam8 small tensors', op='adam8', form='tensors', numel=2049, tensors=7, dtype='float32'),
        # one flat fp32 parameter of 16 Mi elements
        dict(name='adam8 flat 16Mi', op='adam8', form='tensors', numel=16 << 20, tensors=1, dtype='float32'),
        # a chunk set of odd tensors, fp16 gradients under a loss scale, no clipping
        dict(name='adam8 chunks fp16', op='adam8', form='chunks', hidden=1000, ffn=2999, layers=9, vocab=20011, chunk=17000003,
             dtype='float16', loss_scale=1024.0, max_norm=0.0),
        # OPT-1.3B: 11 chunks of 128 Mi, bf16 gradients, clipped to norm 1
        dict(name='adam8 chunks bf16 1.3B', op='adam8', form='chunks', hidden=2048, ffn=8192, layers=24, vocab=50272, chunk=128 << 20,
             dtype='bfloat16', loss_scale=1.0, max_norm=1.0),
        # one token through a norm of OPT-1.3B
        dict(name='layer_norm 1 token', op='layer_norm', rows=1, cols=2048, dtype='bfloat16', train=False),
        # a ragged micro-batch at an odd width
        dict(name='layer_norm train odd fp16', op='layer_norm', rows=2047, cols=769, dtype='float16', train=True),
        # a micro-batch of 4 x 2048 tokens, OPT-1.3B
        dict(name='layer_norm train bf16', op='layer_norm', rows=8192, cols=2048, dtype='bfloat16', train=True),
        # fp32 training at the width of LLaMA-7B
        dict(name='layer_norm train fp32', op='layer_norm', rows=16384, cols=4096, dtype='float32', train=True),
        # the tokens of one step of eight sequences being generated
        dict(name='embedding 8 tokens', op='embedding', tokens=8, vocab=50272, cols=2048, dtype='bfloat16', scale=1.0, padded=0.0,
             train=False),
        # GPT-2's table, a short odd micro-batch, a third of it padding
        dict(name='embedding train padded fp16', op='embedding', tokens=1021, vocab=50257, cols=768, dtype='float16', scale=1.0,
             padded=0.33, train=True),
        # OPT-1.3B's table, 8 x 2048 tokens, embeddings scaled by the root of the width
        dict(name='embedding train bf16', op='embedding', tokens=16384, vocab=50272, cols=2048, dtype='bfloat16', scale=2048 ** 0.5,
             padded=0.0, train=True),
        # LLaMA-7B's table in fp32
        dict(name='embedding train fp32', op='embedding', tokens=8191, vocab=32000, cols=4096, dtype='float32', scale=1.0, padded=0.1,
             train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(sorted(DTYPES))
    op = rng.choice(['adam8 tensors', 'adam8 chunks', 'layer_norm', 'layer_norm', 'embedding', 'embedding'])
    if op == 'adam8 tensors':
        tensors = rng.randint(1, 20)
        return dict(op='adam8', form='tensors', numel=_log_int(rng, 1, (16 << 20) // tensors), tensors=tensors, dtype='float32')
    if op == 'adam8 chunks':
        dtype = rng.choice(['float16', 'bfloat16'])
        hidden, ffn, vocab = _log_int(rng, 64, 2048), _log_int(rng, 64, 8192), _log_int(rng, 100, 50272)
        case = dict(op='adam8', form='chunks', hidden=hidden, ffn=ffn, layers=rng.randint(1, 12), vocab=vocab, chunk=0, dtype=dtype,
                    loss_scale=1024.0 if dtype == 'float16' else 1.0, max_norm=1.0 if dtype == 'bfloat16' else rng.choice([0.0, 1.0]))
        sizes = [math.prod(s) for s in _chunk_shapes(case)]
        least = max(max(sizes), sum(sizes) // 6)
        return dict(case, chunk=least + rng.randint(0, least))
    if op == 'layer_norm':
        cols = _log_int(rng, 16, 4096)
        cols = cols // 8 * 8 if rng.random() < 0.6 else cols
        return dict(op='layer_norm', rows=_log_int(rng, 1, 16384), cols=cols, dtype=dtype, train=rng.random() < 0.7)
    cols = _log_int(rng, 16, 4096)
    cols = cols // 8 * 8 if rng.random() < 0.6 else cols
    return dict(op='embedding', tokens=_log_int(rng, 1, 16384), vocab=_log_int(rng, 100, 50272), cols=cols, dtype=dtype,
                scale=rng.choice([1.0, round(cols ** 0.5, 6)]), padded=rng.choice([0.0, 0.0, 0.5]), train=rng.random() < 0.7)


def _tensor_sizes(case):
    """Tensors around ``numel`` elements, no two alike."""
    n = case['numel']
    return [max(1, n - (i * n) // (2 * case['tensors']) + (i & 1)) for i in range(case['tensors'])]


def _chunk_shapes(case):
    """The tensors of a decoder: table, per layer four square and two ffn matrices with their biases and two norms."""
    h, f = case['hidden'], case['ffn']
    layer = [(h, h), (h, )] * 4 + [(h, ), (h, ), (f, h), (f, ), (h, f), (h, ), (h, ), (h, )]
    return [(case['vocab'], h)] + layer * case['layers'] + [(h, ), (h, )]


def _packed(case):
    """The greedy packing into chunks: number of chunks and elements used in each."""
    used = []
    for shape in _chunk_shapes(case):
        n = math.prod(shape)
        if not used or case['chunk'] - used[-1] < n:
            used.append(0)
        used[-1] += n
    return used


def work(case):
    es = ESIZE[case['dtype']]
    if case['op'] == 'adam8':
        if case['form'] == 'tensors':
            n, per = sum(_tensor_sizes(case)), 4 + 8 + 4 + 4    # gradient, parameter, codes, the state returned in 16 bits
        else:
            n, per = sum(_packed(case)), 2 * es + 8 + 4 + 4     # gradient in, low-precision copy out, as above
        return dict(bytes=n * per, flops=n * 40)
    if case['op'] == 'layer_norm':
        n = case['rows'] * case['cols']
        if not case['train']:
            return dict(bytes=2 * n * es + 2 * case['cols'] * es, flops=8 * n)
        return dict(bytes=4 * n * es + 4 * case['cols'] * es, flops=22 * n)    # x, dy in; y, dx out
    n, table = case['tokens'] * case['cols'], case['vocab'] * case['cols']
    rows = min(case['tokens'], case['vocab']) * case['cols']
    if not case['train']:
        return dict(bytes=(rows + n) * es + 8 * case['tokens'], flops=n)
    return dict(bytes=(rows + 2 * n + table) * es + 8 * case['tokens'], flops=2 * n)


# --------------------------------------------------------------------------------------------------------- the 8-bit code


def _blocks(x):
    """[rows, n] as [rows, blocks, 256], the end filled with zeros."""
    pad = -x.shape[1] % BLOCK
    return torch.nn.functional.pad(x, (0, pad)).view(x.shape[0], -1, BLOCK)


def _exponent(x):
    """E of every block of [rows, blocks, 256]: magnitudes whose fraction is above 1.75 take the next exponent."""
    return (x.abs().amax(2, keepdim=True).view(torch.int32) + 0x1FFFFF) >> 23


def _pow2(e):
    """2^e in 32 bits, for the exponents of ordinary numbers."""
    return ((e + 127) << 23).view(torch.float32)


def _mix(x):
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _dither(first, rows, blocks, step, device):
    """20 bits per element of the buffers ``first`` and up: one 32-bit word per four elements, turned by 8 bits from one to the
    next.  A buffer goes by its place among the parameters, or among the chunks."""
    salt = torch.arange(first, first + rows, device=device).view(-1, 1, 1, 1)
    block = torch.arange(blocks, device=device).view(1, -1, 1, 1)
    lane = torch.arange(64, device=device).view(1, 1, -1, 1)
    key = _mix(block ^ _mix((salt * 0x9E3779B9 + step) & 0xFFFFFFFF))
    word = _mix((key + lane * 0x9E3779B9) & 0xFFFFFFFF)
    turn = torch.arange(4, device=device).view(1, 1, 1, -1) * 8
    turned = ((word >> turn) | (word << (32 - turn))) & 0xFFFFFFFF
    return (turned >> 12).view(rows, blocks, BLOCK).to(torch.int32)


def _round_avg(m):
    """exp_avg [rows, blocks, 256] -> (codes, E)."""
    e = _exponent(m)
    return (m * _pow2(135 - e)).to(torch.float8_e4m3fn), e


def _round_sq(v, dither):
    e = _exponent(v)
    bits = (v * _pow2(31 - e)).view(torch.int32)
    return torch.maximum((bits + dither) >> 20, (bits != 0).to(torch.int32)).to(torch.uint8), e


def _value_avg(code, e):
    return code.to(torch.float32) * _pow2(e - 135)


def _value_sq(code, e):
    return (code.to(torch.int32) << 20).view(torch.float32) * _pow2(e - 31)


# ---------------------------------------------------------------------------------------------------------------- inputs


def _moments(rows, n, used, grad, gen):
    """Moments of a run under way, as the codes hold them: exp_avg a tenth of the root of exp_avg_sq, that one of the size of
    the gradients this run has seen, ``grad`` and up, different from block to block."""
    size = grad * 10.0 ** torch.rand(rows, (n + BLOCK - 1) // BLOCK, 1, generator=gen, device='cuda')
    m = torch.randn(rows, size.shape[1], BLOCK, generator=gen, device='cuda') * size * 0.1
    v = (torch.rand(rows, size.shape[1], BLOCK, generator=gen, device='cuda') + 1).mul_(size).square_()
    outside = torch.arange(size.shape[1] * BLOCK, device='cuda').view(1, -1) >= torch.tensor(used, device='cuda').view(-1, 1)
    m.view(rows, -1).masked_fill_(outside, 0.0)
    v.view(rows, -1).masked_fill_(outside, 0.0)
    half = torch.full((1, ), 1 << 19, dtype=torch.int32, device='cuda')
    return _round_avg(m) + _round_sq(v, half)


def _prepare_tensors(case, gen):
    sizes = _tensor_sizes(case)
    params = [torch.randn(n, generator=gen, device='cuda') * 0.02 for n in sizes]
    grads = [torch.randn(n, generator=gen, device='cuda') * 1e-3 for n in sizes]
    moments = [_moments(1, n, [n], 1e-3, gen) for n in sizes]
    state = dict(case=case, step=FIRST_STEP, params=params, grads=grads, moments=moments)
    if own:
        import elixir_amd as ea
        state['params'] = [torch.nn.Parameter(p) for p in params]
        for p, g in zip(state['params'], grads):
            p.grad = g
        opt = state['opt'] = ea.HybridAdam(state['params'], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=8)
        saved = {
            i: dict(step=FIRST_STEP, exp_avg=_value_avg(mc, me).reshape(-1)[:n], exp_avg_sq=_value_sq(vc, ve).reshape(-1)[:n])
            for i, (n, (mc, me, vc, ve)) in enumerate(zip(sizes, moments))
        }
        opt.load_state_dict(dict(state=saved, param_groups=opt.state_dict()['param_groups']))
    return state


def _prepare_chunks(case, gen):
    dtype, size = DTYPES[case['dtype']], case['chunk']
    used = _packed(case)
    rows = len(used)
    inside = torch.arange(size, device='cuda').view(1, -1) < torch.tensor(used, device='cuda').view(-1, 1)
    master = torch.randn(rows, size, generator=gen, device='cuda').mul_(0.02).mul_(inside)
    grads = torch.randn(rows, size, generator=gen, device='cuda').mul_(1e-2 * case['loss_scale']).mul_(inside).to(dtype)
    clip = max(1.0, 1e-2 * sum(used) ** 0.5 / case['max_norm']) if case['max_norm'] > 0 else 1.0
    moments = _moments(rows, size, used, 1e-2 / clip, gen)
    del inside
    state = dict(case=case, step=FIRST_STEP, master=master, grads=grads, moments=moments)
    if own:
        import elixir_amd as ea
        # a tensor that is longer than a chunk is cut to it, as the rows above are
        named = [('t%d' % i, shape if math.prod(shape) <= size else (size, )) for i, shape in enumerate(_chunk_shapes(case))]
        module = ea.ElixirModule(dict(named), ea.greedy_search([(n, math.prod(s)) for n, s in named], size, dtype), dtype=dtype)
        inner = ea.HybridAdam(list(module.parameters()), lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=8)
        opt = ea.ElixirOptimizer(module, inner, initial_scale=case['loss_scale'], max_norm=case['max_norm'])
        mc, me, vc, ve = moments
        m, v = _value_avg(mc, me).view(rows, -1), _value_sq(vc, ve).view(rows, -1)
        place = {chunk.paired_chunk: i for i, chunk in enumerate(module.param_chunks)}
        for chunk, i in place.items():
            chunk.shard.copy_(master[i])
        saved = {}
        for i, p in enumerate(inner.param_groups[0]['params']):
            row, (begin, end) = place[opt.param_to_optim_chunk[p]], opt.param_to_range[p]
            saved[i] = dict(step=FIRST_STEP, exp_avg=m[row, begin:end], exp_avg_sq=v[row, begin:end])
        inner.load_state_dict(dict(state=saved, param_groups=inner.state_dict()['param_groups']))
        state.update(module=module, opt=opt, payloads=list(grads))
    return state


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    if case['op'] == 'adam8':
        return _prepare_tensors(case, gen) if case['form'] == 'tensors' else _prepare_chunks(case, gen)
    dtype, cols = DTYPES[case['dtype']], case['cols']
    if case['op'] == 'layer_norm':
        # rows of different means and sizes, weights around one: activations between two blocks of a decoder
        shape = (case['rows'], cols)
        spread = 0.5 + 2 * torch.rand(case['rows'], 1, generator=gen, device='cuda')
        x = torch.randn(shape, generator=gen, device='cuda') * spread + torch.randn(case['rows'], 1, generator=gen, device='cuda')
        weight = 1 + 0.1 * torch.randn(cols, generator=gen, device='cuda')
        bias = 0.1 * torch.randn(cols, generator=gen, device='cuda')
        state = dict(case=case, x=x.to(dtype), weight=weight.to(dtype), bias=bias.to(dtype))
        if case['train']:
            state['dy'] = (torch.randn(shape, generator=gen, device='cuda') * 1e-2).to(dtype)
            state.update({k: state[k].requires_grad_() for k in ('x', 'weight', 'bias')})
        return state
    tokens, vocab = case['tokens'], case['vocab']
    # few tokens make up most of a text
    index = (torch.rand(tokens, generator=gen, device='cuda') ** 3 * vocab).long().clamp_(max=vocab - 1)
    index[tokens - int(tokens * case['padded']):] = 1
    state = dict(case=case, index=index, table=(torch.randn(vocab, cols, generator=gen, device='cuda') * 0.02).to(dtype),
                 padding=1 if case['padded'] else None)
    if case['train']:
        state['dy'] = (torch.randn(tokens, cols, generator=gen, device='cuda') * 1e-2).to(dtype)
        state['table'].requires_grad_()
    return state


# ----------------------------------------------------------------------------------------------------------- plain forms


def _plain_adam8(p, g, moments, step, scale, first=0):
    """One step over [rows, n], the buffers ``first`` and up: p is updated in place; returns the new (codes, E, codes, E)."""
    rows, n = p.shape
    mc, me, vc, ve = moments
    g = _blocks(g.float())
    g = g / scale if scale != 1.0 else g
    m = _value_avg(mc, me)
    m += (g - m) * (1 - BETAS[0])
    v = _value_sq(vc, ve)
    v = v * BETAS[1] + g * g * (1 - BETAS[1])
    del g
    denom = v.sqrt() / math.sqrt(1 - BETAS[1] ** step) + EPS
    change = (m / denom).view(rows, -1)[:, :n] * (LR / (1 - BETAS[0] ** step))
    p.mul_(1 - LR * DECAY).sub_(change)
    del denom, change
    return _round_avg(m) + _round_sq(v, _dither(first, rows, m.shape[1], step, p.device))


def _states(moments, n):
    mc, me, vc, ve = moments
    rows = mc.shape[0]
    return (list(_value_avg(mc, me).to(torch.bfloat16).view(rows, -1)[:, :n]),
            list(_value_sq(vc, ve).to(torch.bfloat16).view(rows, -1)[:, :n]))


def _run_adam8(state):
    case = state['case']
    if case['form'] == 'tensors':
        if own:
            opt, params = state['opt'], state['params']
            opt.step()
            moments = [opt.read_moments(p, torch.bfloat16) for p in params]
            return dict(params=[p.detach() for p in params], exp_avg=[m for m, _ in moments], exp_avg_sq=[v for _, v in moments])
        state['step'] += 1
        state['moments'] = [
            _plain_adam8(p.view(1, -1), g.view(1, -1), mo, state['step'], 1.0, i)
            for i, (p, g, mo) in enumerate(zip(state['params'], state['grads'], state['moments']))
        ]
        moments = [_states(mo, p.numel()) for p, mo in zip(state['params'], state['moments'])]
        return dict(params=state['params'], exp_avg=[m[0] for m, _ in moments], exp_avg_sq=[v[0] for _, v in moments])
    if own:
        module, opt = state['module'], state['opt']
        from elixir_amd.chunk import land_chunks
        land_chunks(module.param_chunks, state['payloads'])
        opt.mark_gradients_scaled()
        opt.step()
        moments = [opt.optim.binding.read_moments(c.paired_chunk, torch.bfloat16) for c in module.param_chunks]
        return dict(master=[c.paired_chunk.shard for c in module.param_chunks], lowp=[c.shard for c in module.param_chunks],
                    exp_avg=[m for m, _ in moments], exp_avg_sq=[v for _, v in moments])
    state['step'] += 1
    master, grads = state['master'], state['grads']
    norm = grads.float().square_().sum(dtype=torch.float64).sqrt().item()    # not finite: the step would be skipped
    scale = case['loss_scale']
    if case['max_norm'] > 0:
        scale *= max(1.0, (norm / scale + 1e-6) / case['max_norm'])
    if math.isfinite(norm):
        state['moments'] = _plain_adam8(master, grads, state['moments'], state['step'], scale)
    exp_avg, exp_avg_sq = _states(state['moments'], master.shape[1])
    return dict(master=list(master), lowp=list(master.to(grads.dtype)), exp_avg=exp_avg, exp_avg_sq=exp_avg_sq)


def _run_layer_norm(state):
    case, x, weight, bias = state['case'], state['x'], state['weight'], state['bias']
    if own:
        import elixir_amd as ea
        y = ea.layer_norm(x, weight, bias)
        if not case['train']:
            return dict(y=y)
        dx, dweight, dbias = torch.autograd.grad(y, (x, weight, bias), state['dy'])
        return dict(y=y.detach(), dx=dx, dweight=dweight, dbias=dbias)
    with torch.no_grad():
        dtype = x.dtype
        x, w = x.float(), weight.float()
        centred = x - x.mean(1, keepdim=True)
        rstd = (centred.square().mean(1, keepdim=True) + 1e-5).rsqrt()
        xhat = centred * rstd
        y = (xhat * w + bias.float()).to(dtype)
        if not case['train']:
            return dict(y=y)
        dy = state['dy'].float()
        dxhat = dy * w
        dx = (dxhat - dxhat.mean(1, keepdim=True) - xhat * (dxhat * xhat).mean(1, keepdim=True)) * rstd
        return dict(y=y, dx=dx.to(dtype), dweight=(dy * xhat).sum(0, dtype=torch.float64).to(dtype),
                    dbias=dy.sum(0, dtype=torch.float64).to(dtype))


def _run_embedding(state):
    case, index, table = state['case'], state['index'], state['table']
    if own:
        import elixir_amd as ea
        y = ea.embedding(index, table, padding_idx=state['padding'], scale=case['scale'])
        if not case['train']:
            return dict(y=y)
        return dict(y=y.detach(), dtable=torch.autograd.grad(y, table, state['dy'])[0])
    with torch.no_grad():
        y = (table[index].float() * case['scale']).to(table.dtype)
        if not case['train']:
            return dict(y=y)
        dy = state['dy'].double() * case['scale']
        if state['padding'] is not None:
            dy[index == state['padding']] = 0.0
        dtable = torch.zeros(table.shape, dtype=torch.float64, device=table.device).index_add_(0, index, dy)
        return dict(y=y, dtable=dtable.to(table.dtype))


def run(state):
    return dict(adam8=_run_adam8, layer_norm=_run_layer_norm, embedding=_run_embedding)[state['case']['op']](state)


# --------------------------------------------------------------------------------------------------------------- 64 bits


def _exact_code(x, largest_power, mantissa_floor, dither):
    """x [blocks, 256] in 64 bits as a code with three mantissa bits holds it: quanta of an eighth of the power of two below,
    none under ``mantissa_floor`` binades below the largest; ``dither`` None rounds to nearest even."""
    _, e = torch.frexp(x.abs().clamp_min(5e-324))
    quantum = torch.exp2((torch.maximum(e - 1, largest_power - mantissa_floor) - 3).double())
    if dither is None:
        return (x / quantum).round() * quantum
    up = torch.floor(x / quantum + dither.double() * 2.0 ** -20)
    return torch.maximum(up, (x > 0).double()) * quantum


def _exact_step(p, g, m, v, step, salt):
    """One tensor in 64 bits, from the definition: Kingma and Ba's moments, decoupled decay, then the codes of the state."""
    n = p.numel()
    p, g, m, v = p.double(), g.double(), m.double(), v.double()
    b1, b2 = BETAS
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    p = p * (1 - LR * DECAY) - LR * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)) ** 0.5 + EPS)
    fill = -n % BLOCK
    m = torch.cat([m, m.new_zeros(fill)]).view(-1, BLOCK)
    v = torch.cat([v, v.new_zeros(fill)]).view(-1, BLOCK)

    def top(x):
        f, e = torch.frexp(x.abs().amax(1, keepdim=True))
        return e - 1 + (f > 0.875).int()

    dither = _dither(salt, 1, m.shape[0], step, p.device)[0]
    m = _exact_code(m, top(m), 14, None)
    v = _exact_code(v, top(v), 30, dither)
    return p, m.view(-1)[:n], v.view(-1)[:n]


def exact(case, seed):
    state = prepare(case, seed)
    step = FIRST_STEP + 1
    if case['op'] == 'adam8' and case['form'] == 'tensors':
        values = [(_value_avg(mc, me).reshape(-1), _value_sq(vc, ve).reshape(-1)) for mc, me, vc, ve in state['moments']]
        done = [_exact_step(p, g, m[:p.numel()], v[:p.numel()], step, i)
                for i, (p, g, (m, v)) in enumerate(zip(state['params'], state['grads'], values))]
        return dict(params=[d[0] for d in done], exp_avg=[d[1] for d in done], exp_avg_sq=[d[2] for d in done])
    if case['op'] == 'adam8':
        size, scale = case['chunk'], case['loss_scale']
        if case['max_norm'] > 0:
            norm = sum(g.double().square().sum().item() for g in state['grads']) ** 0.5
            scale *= max(1.0, (norm / scale + 1e-6) / case['max_norm'])
        mc, me, vc, ve = state['moments']
        m, v = _value_avg(mc, me).view(len(mc), -1), _value_sq(vc, ve).view(len(mc), -1)
        done = [_exact_step(state['master'][i], state['grads'][i].double() / scale, m[i, :size], v[i, :size], step, i)
                for i in range(len(mc))]
        return dict(master=[d[0] for d in done], lowp=[d[0] for d in done], exp_avg=[d[1] for d in done],
                    exp_avg_sq=[d[2] for d in done])
    if case['op'] == 'layer_norm':
        x, w, b = (state[k].detach().double() for k in ('x', 'weight', 'bias'))
        n = x.shape[1]
        mean = x.sum(1, keepdim=True) / n
        var = ((x - mean) ** 2).sum(1, keepdim=True) / n
        std = torch.sqrt(var + 1e-5)
        y = (x - mean) / std * w + b
        if not case['train']:
            return dict(y=y)
        dy = state['dy'].double()
        h = (x - mean) / std
        t = dy * w
        dx = (n * t - t.sum(1, keepdim=True) - h * (t * h).sum(1, keepdim=True)) / (n * std)
        return dict(y=y, dx=dx, dweight=torch.einsum('rc,rc->c', dy, h), dbias=dy.sum(0))
    table, index = state['table'].detach().double(), state['index']
    y = torch.index_select(table, 0, index) * case['scale']
    if not case['train']:
        return dict(y=y)
    keep = torch.ones(case['tokens'], dtype=torch.float64, device='cuda')
    if state['padding'] is not None:
        keep = (index != state['padding']).double()
    dtable = torch.zeros_like(table)
    dtable.index_put_((index, ), state['dy'].double() * (keep * case['scale'])[:, None], accumulate=True)
    return dict(y=y, dtable=dtable)
