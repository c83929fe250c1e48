"""layer_norm, embedding and their modules without a GPU: what they refuse, what the modules leave to torch, and the swap."""
import copy
import pickle

import pytest
import torch
from torch import nn
from torch.fx.experimental.proxy_tensor import make_fx

import elixir_amd as ea
from elixir_amd import _abi, _ops_abi, _torch_ext
from elixir_amd.fused_ops import fuse_modules


def test_functions_refuse_what_they_cannot_take():
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match='GPU'):
        ea.layer_norm(x, w, w)
    with pytest.raises(ValueError, match='shape'):
        ea.layer_norm(x, torch.ones(4))
    with pytest.raises(ValueError, match='bias has shape'):
        ea.layer_norm(x, w, torch.ones(1, 8))
    with pytest.raises(ValueError, match='layer_norm over'):
        ea.layer_norm(x, normalized_shape=(2, 8))
    with pytest.raises(ValueError, match='layer_norm over'):
        ea.layer_norm(torch.tensor(1.0))
    table = torch.zeros(10, 4)
    with pytest.raises(RuntimeError, match='GPU'):
        ea.embedding(torch.zeros(3, dtype=torch.int64), table)
    with pytest.raises(TypeError, match='int64 or int32'):
        ea.embedding(torch.zeros(3), table)
    with pytest.raises(ValueError, match='two dimensions'):
        ea.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(4))


def test_the_extension_carries_its_stamp(monkeypatch):
    from elixir_amd import build as B
    assert _torch_ext.built_stamp(_torch_ext.LIB_PATH) == _torch_ext.stamp() and _torch_ext.stamp() in _torch_ext.load().stamp
    assert _torch_ext.built_stamp('/nowhere') == ''
    monkeypatch.setattr(_torch_ext, '_ext', None)
    monkeypatch.setattr(_torch_ext, 'stamp', lambda: 'other')
    with pytest.raises(RuntimeError, match='built from something else'):
        _torch_ext.load()
    assert B.is_stale()


def test_launches_refuse_what_they_cannot_run():
    at = 1 << 20
    F32, F16 = _abi.ELX_F32, _abi.ELX_F16

    def refused(code, call, *args):
        with pytest.raises(_abi.ElxError) as e:
            call(*args)
        assert e.value.code == code

    fwd = _ops_abi.layer_norm_fwd
    refused(_abi.ELX_E_NULL, fwd, 0, at, at, at, at, at, 4, 8, 8, 1e-5, F32, 0)
    refused(_abi.ELX_E_NULL, fwd, at, at, at, 0, at, at, 4, 8, 8, 1e-5, F32, 0)
    refused(_abi.ELX_E_DTYPE, fwd, at, at, at, at, at, at, 4, 8, 8, 1e-5, 5, 0)
    refused(_abi.ELX_E_SIZE, fwd, at, at, at, at, at, at, 0, 8, 8, 1e-5, F32, 0)
    refused(_abi.ELX_E_SIZE, fwd, at, at, at, at, at, at, 4, 0, 8, 1e-5, F32, 0)
    refused(_abi.ELX_E_SIZE, fwd, at, at, at, at, at, at, 4, 16385, 16385, 1e-5, F32, 0)
    refused(_abi.ELX_E_RANGE, fwd, at, at, at, at, at, at, 4, 8, 7, 1e-5, F32, 0)
    refused(_abi.ELX_E_ALIGN, fwd, at + 1, at, at, at, at, at, 4, 8, 8, 1e-5, F16, 0)
    refused(_abi.ELX_E_ALIGN, fwd, at, at, at, at, at + 2, at, 4, 8, 8, 1e-5, F16, 0)
    bwd, ws = _ops_abi.layer_norm_bwd, _ops_abi.layer_norm_bwd_workspace(4, 8)
    assert ws >= 2 * 8 * 4
    refused(_abi.ELX_E_NULL, bwd, 0, at, at, at, at, at, at, at, at, ws, 4, 8, 8, 8, F32, 0)
    refused(_abi.ELX_E_NULL, bwd, at, at, at, 0, at, at, at, at, at, ws, 4, 8, 8, 8, F32, 0)
    refused(_abi.ELX_E_NULL, bwd, at, at, at, at, at, 0, 0, 0, at, ws, 4, 8, 8, 8, F32, 0)
    refused(_abi.ELX_E_NULL, bwd, at, at, at, at, at, at, at, at, 0, ws, 4, 8, 8, 8, F32, 0)
    refused(_abi.ELX_E_SIZE, bwd, at, at, at, at, at, at, at, at, at, ws - 1, 4, 8, 8, 8, F32, 0)
    refused(_abi.ELX_E_SIZE, bwd, at, at, at, at, at, at, at, at, at, 1 << 40, 4, 16385, 16385, 16385, F32, 0)
    refused(_abi.ELX_E_RANGE, bwd, at, at, at, at, at, at, at, at, at, ws, 4, 8, 7, 8, F32, 0)
    refused(_abi.ELX_E_ALIGN, bwd, at, at + 2, at, at, at, at, at, at, at, ws, 4, 8, 8, 8, F32, 0)
    look = _ops_abi.embedding_fwd
    refused(_abi.ELX_E_NULL, look, 0, 8, 4, at, 10, 8, 1.0, at, F32, 0)
    refused(_abi.ELX_E_DTYPE, look, at, 2, 4, at, 10, 8, 1.0, at, F32, 0)
    refused(_abi.ELX_E_SIZE, look, at, 8, 0, at, 10, 8, 1.0, at, F32, 0)
    refused(_abi.ELX_E_SIZE, look, at, 8, 4, at, 0, 8, 1.0, at, F32, 0)
    refused(_abi.ELX_E_SIZE, look, at, 8, (1 << 26) + 1, at, 10, 8, 1.0, at, F32, 0)
    refused(_abi.ELX_E_ALIGN, look, at + 4, 8, 4, at, 10, 8, 1.0, at, F32, 0)
    grad, ws = _ops_abi.embedding_bwd, _ops_abi.embedding_bwd_workspace(4, 10, 8)
    assert ws > 0 and _ops_abi.embedding_bwd_workspace(0, 10, 8) == 0
    refused(_abi.ELX_E_NULL, grad, at, 8, 4, at, 8, at, 10, 8, 1.0, -1, 0, ws, F32, 0)
    refused(_abi.ELX_E_SIZE, grad, at, 8, 4, at, 8, at, 10, 8, 1.0, -1, at, ws - 1, F32, 0)
    refused(_abi.ELX_E_RANGE, grad, at, 8, 4, at, 7, at, 10, 8, 1.0, -1, at, ws, F32, 0)
    refused(_abi.ELX_E_ALIGN, grad, at, 8, 4, at + 1, 8, at, 10, 8, 1.0, -1, at, ws, F16, 0)
    refused(_abi.ELX_E_ALIGN, grad, at, 8, 4, at, 8, at, 10, 8, 1.0, -1, at + 8, ws, F16, 0)


def test_rows_are_found_in_place_or_copied():
    _rows = _torch_ext.load().rows_of
    base = torch.arange(240.).view(4, 5, 12)
    for x, cols, stride in ((base, 12, 12), (base[..., :8], 8, 12), (base[:, 2], 12, 60), (base[1], 12, 12), (base[::2, :, 3:7], 4, None),
                            (base.transpose(0, 1), 12, None), (base[..., ::2], 6, None), (base[0, 0].expand(3, 12), 12, None),
                            (base[:, :1, :1], 1, 60), (base[:1, :, 2:3], 1, 12), (base[0, 0, :7], 7, 7)):
        got, step = _rows(x, cols)
        assert got.data_ptr() == x.data_ptr() if stride is not None else got.is_contiguous() and got.data_ptr() != x.data_ptr()
        assert step == (cols if stride is None else stride)
        flat = torch.as_strided(got, (x.numel() // cols, cols), (step, 1)) if x.numel() else got
        assert torch.equal(flat.reshape(x.shape), x)


class Net(nn.Module):

    def __init__(self):
        super().__init__()
        self.emb = nn.Embedding(20, 16, padding_idx=3)
        self.norm = nn.LayerNorm(16)
        self.plain = nn.LayerNorm(16, elementwise_affine=False)
        self.group = nn.GroupNorm(2, 16)

    def forward(self, x):
        return self.plain(self.norm(self.emb(x)))


def test_the_swap_keeps_objects_parameters_and_results():
    torch.manual_seed(0)
    net = Net()
    x = torch.tensor([[1, 3, 5], [19, 0, 1]])
    want = net(x)
    params, norm = dict(net.named_parameters()), net.norm
    sub = type('Sub', (nn.LayerNorm, ), {})(16)
    net.sub = sub
    assert fuse_modules(net) == 3
    assert type(net.emb) is ea.FusedEmbedding and type(net.norm) is ea.FusedLayerNorm and net.norm is norm and type(net.sub) is not ea.FusedLayerNorm
    assert all(dict(net.named_parameters())[n] is p for n, p in params.items())
    assert torch.equal(net(x), want)    # on the CPU: torch's own
    assert fuse_modules(net) == 0
    del net.sub
    for twin in (copy.deepcopy(net), pickle.loads(pickle.dumps(net))):
        assert type(twin.norm) is ea.FusedLayerNorm and torch.equal(twin(x), want)
    net(x).sum().backward()
    assert net.emb.weight.grad[3].abs().sum() == 0 and net.emb.weight.grad[1].abs().sum() >= 0


def test_elixir_module_swaps_only_when_asked():
    for kw, fused in ((dict(), False), (dict(use_fused_kernels=True), False), (dict(fused_ops=True), True)):
        net = Net()
        named = [(n, p.numel()) for n, p in net.named_parameters()]
        module = ea.ElixirModule(net, ea.greedy_search(named, 400, torch.float32), dtype=torch.float32, **kw)
        assert (type(net.norm) is ea.FusedLayerNorm) == fused and module.fused_ops == fused
    shapes = {'a': (3, 4)}
    assert ea.ElixirModule(shapes, ea.greedy_search([('a', 12)], 16, torch.float32), fused_ops=True).fused_ops


def test_scale_of_the_embedding_module():
    emb = ea.FusedEmbedding(10, 4, scale=2.0)
    assert torch.equal(emb(torch.tensor([3])), emb.weight[3:4] * 2)
    emb = ea.FusedEmbedding(10, 4, max_norm=0.1)
    assert emb(torch.tensor([3])).norm() <= 0.1001


def test_transforms_that_see_only_the_allocations_are_refused():
    """A tangent must not be dropped and a trace must not record an empty tensor in place of the result."""
    x, w, index = torch.randn(3, 8), torch.randn(8), torch.tensor([1, 2])
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            ea.layer_norm(dual, w)
        with pytest.raises(NotImplementedError, match='forward-mode'):
            ea.layer_norm(x, torch.autograd.forward_ad.make_dual(w, w))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            ea.embedding(index, dual)
    for call in (lambda: torch.jit.trace(lambda t: ea.layer_norm(t, w), x, check_trace=False),
                 lambda: make_fx(lambda t: ea.layer_norm(t, w))(x), lambda: make_fx(lambda t: ea.embedding(index, t))(x)):
        with pytest.raises(NotImplementedError, match='traced'):
            call()
