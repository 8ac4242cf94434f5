"""A layer and a weighted return keep for their backward what the wanted gradients read, and nothing else: the rest may
change in place."""
import pytest
import torch

from odie_amd.linear import linear
from odie_amd.mixture import combine, expert_order

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('grouped', (False, True))
@pytest.mark.parametrize('activation', ('none', 'gelu'))
def test_tensors_that_no_gradient_reads_may_change(activation, grouped):
    generator = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randn(90, 24, generator=generator, device='cuda')
    w = torch.randn(*((3,) if grouped else ()), 16, 24, generator=generator, device='cuda')
    b = torch.randn(w.shape[:-1], generator=generator, device='cuda')
    dy = torch.randn(90, 16, generator=generator, device='cuda')
    offsets = torch.tensor([0, 30, 50, 90], dtype=torch.int32, device='cuda') if grouped else None

    def gradient(wanted, change):
        leaves = {name: value.clone().requires_grad_(name == wanted) for name, value in (('x', x), ('w', w), ('b', b))}
        y = linear(leaves['x'], leaves['w'], leaves['b'], activation=activation, offsets=offsets)
        for name in change:
            with torch.no_grad():
                leaves[name].zero_()
        return torch.autograd.grad(y, leaves[wanted], dy)[0]

    for wanted, unread, read in (('x', ('b', 'x'), 'w'), ('w', ('b', 'w'), 'x'), ('b', ('x', 'w', 'b'), None)):
        assert torch.equal(gradient(wanted, unread), gradient(wanted, ()))
        if read:
            with pytest.raises(RuntimeError, match='modified by an inplace operation'):
                gradient(wanted, (read,))


def test_weights_of_a_return_that_no_gradient_reads_may_change():
    generator = torch.Generator(device='cuda').manual_seed(2)
    order = expert_order(torch.arange(60, device='cuda').view(30, 2) % 7, 7)
    rows = torch.randn(60, 12, generator=generator, device='cuda')
    weights = torch.rand(30, 2, generator=generator, device='cuda')
    dy = torch.randn(30, 12, generator=generator, device='cuda')
    for change in (False, True):
        leaf = weights.clone().requires_grad_(True)
        y = combine(rows, order, leaf)
        if change:
            with torch.no_grad():
                leaf.zero_()
        got, = torch.autograd.grad(y, leaf, dy)
        if not change:
            expected = got
        assert torch.equal(got, expected)
    leaf, moving = rows.clone().requires_grad_(True), weights.clone()
    y = combine(leaf, order, moving)
    moving.zero_()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(y, leaf, dy)


def test_offsets_that_no_gradient_reads_may_change():
    x, w = torch.ones(8, 16, device='cuda'), torch.ones(2, 24, 16, device='cuda')
    residual = torch.zeros(8, 24, device='cuda', requires_grad=True)
    offsets = torch.tensor([0, 3, 8], dtype=torch.int32, device='cuda')
    y = linear(x, w, residual=residual, offsets=offsets)
    offsets.zero_()
    up = torch.randn_like(y)
    assert torch.equal(torch.autograd.grad(y, residual, up)[0], up)
