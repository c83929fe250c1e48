"""Device memory that a chunked module and its optimizer take from the driver."""
import gc

import pytest
import torch

import elixir_amd as ea

pytestmark = pytest.mark.gpu
MIB = 1 << 20


@pytest.mark.parametrize('state_bits', [8, 32])
@pytest.mark.parametrize('chunks', [1, 4])
def test_the_pool_is_as_large_as_the_state(state_bits, chunks):
    """2^28 elements in fp16: shards 2, master weights 4 and moments 8 bytes each, or 2 and two bytes per block of 256 in 8 bits.
    On top the pool's own slack (256 MiB), and 64 MiB for tables and what the caching allocator rounds up."""
    n, dtype = 1 << 28, torch.float16
    gc.collect()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_reserved()
    named = {f'w{i}': (n // chunks, ) for i in range(chunks)}
    module = ea.ElixirModule(named, ea.greedy_search([(k, n // chunks) for k in named], n // chunks, dtype), dtype=dtype)
    inner = ea.HybridAdam(list(module.parameters()), state_bits=state_bits)
    opt = ea.ElixirOptimizer(module, inner, init_step=True)
    for c in inner.binding.chunks:
        inner.binding.moments(c)
    state = 2 + 4 + (8 if state_bits == 32 else 2 + 2 / 256)
    taken = torch.cuda.memory_reserved() - before
    assert len(module.param_chunks) == chunks
    assert taken <= n * state + 320 * MIB, (taken / MIB, n * state / MIB)    # less where a block was cached before
    del module, inner, opt
    gc.collect()
    torch.cuda.empty_cache()
