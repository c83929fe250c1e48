"""Gradients of ``layer_norm`` and ``embedding`` that are differentiated again, where the inputs of a norm depend on each other: a
norm that two layers share, a weight that is computed from the input, an input computed from the weight.  First and second
derivatives against torch's operators in float64.

Tolerance, derived beforehand: every derivative here is a sum of products of at most 2^8 factors and terms (rows of 32 columns, 5
rows, two norms, a cube), each rounded by 2^-24 of itself, with numbers of the order of the largest result; what is passed on
grows by rstd (at most 2^2 for these rows) at each of the four norms and derivatives of norms of the longest way.  That is
2^-24 * 2^8 * 2^6 = 2^-10 of the largest element at the most; a path that is counted twice is off by a tenth of it and more."""
import pytest
import torch
import torch.nn.functional as F

import elixir_amd as ea

pytestmark = pytest.mark.gpu
DEV = 'cuda'
ROWS, COLS = 5, 32


def shared(norm, x, w, b):
    return norm(torch.tanh(norm(x, w, b)), w, b)


def weight_from_input(norm, x, w, b):
    return norm(x, w + 0.5 * torch.tanh(x).mean(0), b)


def input_from_weight(norm, x, w, b):
    return norm(x * w, w, b)


def recurrent(norm, x, w, b):
    state = torch.zeros_like(x)
    for _ in range(3):
        state = norm(0.5 * state + x, w, b)
    return state


def derivatives(form, norm, leaves, wanted):
    chosen = [t for t, k in zip(leaves, wanted) if k]
    y = form(norm, *leaves)
    first = torch.autograd.grad((y**3).sum(), chosen, create_graph=True)
    second = torch.autograd.grad(sum(t.square().sum() for t in first), chosen, allow_unused=True)
    return [*first, *second]


@pytest.mark.parametrize('form', [shared, weight_from_input, input_from_weight, recurrent])
@pytest.mark.parametrize('wanted', [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 1, 1)])
def test_derivatives_stop_at_the_inputs_of_the_norm(form, wanted):
    g = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(ROWS, COLS, generator=g), 1 + 0.3 * torch.randn(COLS, generator=g), 0.3 * torch.randn(COLS, generator=g)
    got = derivatives(form, lambda *a: ea.layer_norm(*a), [t.to(DEV).requires_grad_() for t in (x, w, b)], wanted)
    want = derivatives(form, lambda x, w, b: F.layer_norm(x, (COLS, ), w, b), [t.double().requires_grad_() for t in (x, w, b)], wanted)
    for a, c in zip(got, want):
        assert (a is None) == (c is None)
        if c is not None:
            assert (a.cpu().double() - c).abs().max() <= 2.0**-10 * c.abs().max()


def test_a_module_that_two_layers_share():
    """The same through FusedLayerNorm and ``backward``, accumulated into the leaves."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(ROWS, COLS, generator=g), 1 + 0.3 * torch.randn(COLS, generator=g)
    grads = []
    for cls, dtype, device in ((ea.FusedLayerNorm, torch.float32, DEV), (torch.nn.LayerNorm, torch.float64, 'cpu')):
        norm = cls(COLS).to(device, dtype)
        norm.weight.data.copy_(w)
        a = x.to(device, dtype).requires_grad_()
        loss = norm(torch.sin(norm(a))).pow(3).sum()
        d, = torch.autograd.grad(loss, a, create_graph=True)
        (loss + d.square().sum()).backward()
        grads.append([a.grad, norm.weight.grad, norm.bias.grad])
    for got, want in zip(*grads):
        assert (got.cpu().double() - want).abs().max() <= 2.0**-10 * want.abs().max()


def test_an_embedding_whose_gradient_is_differentiated_through_its_table():
    """The embedded rows go through a norm whose weight is one of them; the penalty runs through the table twice."""
    g = torch.Generator().manual_seed(2)
    table, index = torch.randn(7, COLS, generator=g), torch.tensor([[0, 3, 3], [6, 2, 0]])
    out = []
    for emb, norm, dtype, device in ((ea.embedding, lambda x, w: ea.layer_norm(x, w), torch.float32, DEV),
                                     (F.embedding, lambda x, w: F.layer_norm(x, (COLS, ), w), torch.float64, 'cpu')):
        t = table.to(device, dtype).requires_grad_()
        y = norm(emb(index.to(device), t), t[3])
        first, = torch.autograd.grad((y**3).sum(), t, create_graph=True)
        out.append((first, torch.autograd.grad(first.square().sum(), t)[0]))
    for got, want in zip(*out):
        assert (got.detach().cpu().double() - want.detach()).abs().max() <= 2.0**-10 * want.abs().max()
