"""A training step as the operators are used together: an ElixirModule with fused_ops, its gradients landing in chunk storage
from inside backward, and the ElixirOptimizer over an 8-bit state."""
import copy

import numpy as np
import pytest
import torch
from torch import nn

import elixir_amd as ea
from helpers import to_np
from oracle import oracle as O
from oracle import state8 as S8
from test_gpu_adam8 import compare_codes, near, segments_of

pytestmark = pytest.mark.gpu
DEV = 'cuda'


class Net(nn.Module):
    """Embedding with padding, two norms, an output projection tied to the embedding."""

    def __init__(self, vocab=211, hidden=72):
        super().__init__()
        self.emb = nn.Embedding(vocab, hidden, padding_idx=0)
        self.norm1 = nn.LayerNorm(hidden)
        self.mix = nn.Linear(hidden, hidden)
        self.norm2 = nn.LayerNorm(hidden, bias=False)

    def forward(self, tokens):
        x = self.norm1(self.emb(tokens))
        x = self.norm2(x + torch.relu(self.mix(x)))
        return x @ self.emb.weight.t()


def loss_of(logits, tokens):
    return nn.functional.cross_entropy(logits.flatten(0, 1).float(), tokens.flatten().long())


def wrap(net, fused, dtype, state_bits, chunk=7000, **kw):
    named = [(n, p.numel()) for n, p in net.named_parameters()]
    module = ea.ElixirModule(net, ea.greedy_search(named, max(chunk, max(s for _, s in named)), dtype), dtype=dtype, fused_ops=fused)
    inner = ea.HybridAdam(net.parameters(), lr=1e-3, weight_decay=0.01, state_bits=state_bits)
    return module, inner, ea.ElixirOptimizer(module, inner, initial_scale=256.0, hysteresis=1, **kw)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('graph', [False, True])
def test_steps_of_a_wrapped_model(oracle, dtype, graph):
    """Each step: forward and backward run on the fused modules, the gradients that land in the shards are within the type's
    rounding of those of torch's modules on the same weights, and the update over the landed gradients has the oracle's codes
    and weights; the next forward sees the refreshed parameters."""
    torch.manual_seed(0)
    net = Net()
    module, inner, opt = wrap(net, True, dtype, 8)
    opt.graph_step = graph
    assert type(net.emb) is ea.FusedEmbedding and type(net.norm1) is ea.FusedLayerNorm and type(net.norm2) is ea.FusedLayerNorm
    twin = Net().to(DEV, dtype)
    scale = opt.loss_scale
    chunks = [pc.paired_chunk for pc in module.param_chunks]
    order = {c: i for i, c in enumerate(inner.binding.chunks)}
    pn = [to_np(c.shard) for c in chunks]
    st = [S8.State8(c.shard_size, order[c]) for c in chunks]
    names = {p: n for n, p in net.named_parameters()}
    gen = torch.Generator().manual_seed(1)
    losses = []
    for step in range(1, 6):
        tokens = torch.randint(0, 211, (5, 33), generator=gen)
        tokens[:, 28:] = 0
        tokens = tokens.to(DEV)
        with torch.no_grad():
            if step > 1:
                module.materialize_params()
            for n, p in twin.named_parameters():
                p.copy_(dict(net.named_parameters())[n])
        twin.zero_grad()
        (loss_of(twin(tokens), tokens) * scale).backward()
        loss = loss_of(module(tokens), tokens)
        opt.backward(loss)
        losses.append(loss.item())
        grads = [to_np(pc.shard) for pc in module.param_chunks]
        for pc in module.param_chunks:
            for p, info in pc.tensors_info.items():
                want = dict(twin.named_parameters())[names[p]].grad.flatten().double()
                got = pc.shard[info.offset:info.end].double()
                # every activation and gradient on the way is rounded to the type by both sides, and a loss of precision in
                # one place spreads: held to 32 half steps of the largest gradient of the tensor
                assert (got - want).abs().max() <= 32 * torch.finfo(dtype).eps / 2 * want.abs().max(), names[p]
        opt.step()
        assert opt.last_step_info['found_inf'] is False
        for i, (pc, c) in enumerate(zip(module.param_chunks, chunks)):
            code = {torch.float16: O.F16, torch.bfloat16: O.BF16, torch.float32: O.F32}[dtype]
            before = pn[i].copy()
            st[i].step(pn[i], grads[i], code, segments_of(opt, inner, c), lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=step,
                       adamw_mode=True, div_scale=scale if scale != 1 else -1.0)
            pn[i] = near(to_np(c.shard), pn[i], before, f'step {step} chunk {i}')
            compare_codes(*inner.binding.moments(c), inner.binding.scales(c), st[i], f'step {step} chunk {i}')
    assert len(losses) == 5 and all(np.isfinite(losses))


def test_the_switches_do_not_touch_each_other():
    """Without fused_ops a model keeps torch's modules and its bits, whatever use_fused_kernels says."""
    runs = []
    for kw in (dict(), dict(use_fused_kernels=True)):
        torch.manual_seed(0)
        net = Net()
        named = [(n, p.numel()) for n, p in net.named_parameters()]
        module = ea.ElixirModule(net, ea.greedy_search(named, 20000, torch.float32), dtype=torch.float32, **kw)
        opt = ea.ElixirOptimizer(module, ea.HybridAdam(net.parameters(), lr=1e-3))
        tokens = torch.arange(60, device=DEV).view(4, 15)
        for _ in range(3):
            opt.backward(loss_of(module(tokens), tokens))
            opt.step()
        runs.append([c.paired_chunk.shard.clone() for c in module.param_chunks])
        assert type(net.norm1) is nn.LayerNorm and type(net.emb) is nn.Embedding
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_resumed_run_continues_with_the_same_bits():
    def data():
        g = torch.Generator().manual_seed(3)
        while True:
            yield torch.randint(0, 211, (4, 20), generator=g).to(DEV)

    def steps(module, opt, batches, n):
        for _ in range(n):
            t = next(batches)
            opt.backward(loss_of(module(t), t))
            opt.step()

    torch.manual_seed(0)
    net = Net()
    module, inner, opt = wrap(net, True, torch.float16, 8, max_norm=1.0)
    batches = data()
    steps(module, opt, batches, 3)
    weights, saved = copy.deepcopy(module.state_dict()), opt.state_dict()
    steps(module, opt, batches, 3)

    torch.manual_seed(9)
    again, inner2, opt2 = wrap(Net(), True, torch.float16, 8, max_norm=1.0)
    again.load_state_dict(weights)
    opt2.load_state_dict(saved)
    batches = data()
    for _ in range(3):
        next(batches)
    steps(again, opt2, batches, 3)
    for a, b in zip(module.param_chunks, again.param_chunks):
        assert torch.equal(a.paired_chunk.shard, b.paired_chunk.shard)
        for x, y in zip(inner.binding.read_moments(a.paired_chunk), inner2.binding.read_moments(b.paired_chunk)):
            assert torch.equal(x, y)
