"""Many gradients of one forward pass at once (``is_grads_batched``, vectorised Jacobians): as torch's modules run them, so do the
fused ones.  Against one backward pass per gradient through the kernels, which the other tests hold.

Tolerance, derived beforehand: both sides sum at most 2^6 numbers in fp32 per element of a result (rows of 48 columns, 6 rows or
tokens) and round about as often again in between; 2^-24 * 2^7 of the largest element, doubled for the two sides."""
import pytest
import torch

import elixir_amd as ea

pytestmark = pytest.mark.gpu
DEV = 'cuda'
COLS = 48


def near(got, want):
    assert got.shape == want.shape and (got - want).abs().max() <= 2.0**-16 * want.abs().max()


def batched(forward, leaves, dys):
    y = forward(*leaves)
    many = torch.autograd.grad(y, leaves, dys, is_grads_batched=True, retain_graph=True)
    ones = [torch.autograd.grad(y, leaves, dy, retain_graph=True) for dy in dys]
    for i, got in enumerate(many):
        near(got, torch.stack([one[i] for one in ones]))


@pytest.mark.parametrize('with_b', [False, True])
def test_layer_norm(with_b):
    g = torch.Generator(device=DEV).manual_seed(0)
    leaves = [torch.randn(*s, generator=g, device=DEV).requires_grad_() for s in ((6, COLS), (COLS, ), (COLS, ))[:3 if with_b else 2]]
    batched(ea.layer_norm, leaves, torch.randn(5, 6, COLS, generator=g, device=DEV))


def test_layer_norm_of_some_inputs():
    g = torch.Generator(device=DEV).manual_seed(1)
    x, w = torch.randn(6, COLS, generator=g, device=DEV), torch.randn(COLS, generator=g, device=DEV)
    dys = torch.randn(5, 6, COLS, generator=g, device=DEV)
    batched(lambda w: ea.layer_norm(x, w), [w.clone().requires_grad_()], dys)
    batched(lambda x: ea.layer_norm(x, w), [x.clone().requires_grad_()], dys)


@pytest.mark.parametrize('padding_idx,scale', [(None, 1.0), (2, 3.0)])
def test_embedding(padding_idx, scale):
    g = torch.Generator(device=DEV).manual_seed(2)
    index = torch.tensor([[0, 2, 2], [8, 5, -1]], device=DEV)
    table = torch.randn(9, COLS, generator=g, device=DEV).requires_grad_()
    batched(lambda t: ea.embedding(index, t, padding_idx=padding_idx, scale=scale).nan_to_num(), [table],
            torch.randn(5, 2, 3, COLS, generator=g, device=DEV))


def test_a_vectorised_jacobian_of_a_fused_model():
    torch.manual_seed(3)
    net = torch.nn.Sequential(torch.nn.LayerNorm(COLS), torch.nn.Linear(COLS, 7)).to(DEV)
    x = torch.randn(4, COLS, device=DEV)
    want = torch.autograd.functional.jacobian(net, x)
    ea.fused_ops.fuse_modules(net)
    assert type(net[0]) is ea.FusedLayerNorm
    near(torch.autograd.functional.jacobian(net, x, vectorize=True), want)


def test_batched_gradients_that_are_differentiated():
    g = torch.Generator(device=DEV).manual_seed(4)
    out = []
    for norm in (lambda x, w: ea.layer_norm(x, w), lambda x, w: torch.nn.functional.layer_norm(x, (COLS, ), w)):
        g.manual_seed(4)
        x, w = (torch.randn(*s, generator=g, device=DEV).requires_grad_() for s in ((6, COLS), (COLS, )))
        dys = torch.randn(5, 6, COLS, generator=g, device=DEV)
        many = torch.autograd.grad(norm(x, w), (x, w), dys, is_grads_batched=True, create_graph=True)
        out.append(torch.autograd.grad(sum(t.square().sum() for t in many), (x, w)))
    for got, want in zip(*out):
        near(got, want)
