"""What the row operators keep for their backward: a change of it in place is noticed, and nothing is kept that no
wanted gradient reads."""
import pytest
import torch

from odie_amd.linear import linear
from odie_amd.mixture import combine, dispatch, expert_order

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('part', ('slots', 'offsets'))
def test_an_order_changed_before_the_backward(part):
    x = torch.randn(6, 8, device='cuda', requires_grad=True)
    rows = torch.randn(12, 8, device='cuda', requires_grad=True)
    weights = torch.rand(6, 2, device='cuda', requires_grad=True)
    for call, leaf in ((lambda order: dispatch(x, order), x), (lambda order: combine(rows, order), rows),
                       (lambda order: combine(rows.detach(), order, weights), weights)):
        order = expert_order(torch.arange(12, device='cuda').view(6, 2) % 5, 5)
        y = call(order)
        getattr(order, part).zero_()
        if part == 'offsets' and leaf is not rows:      # the others' gradients do not read them
            torch.autograd.grad(y, leaf, torch.ones_like(y))
            continue
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            torch.autograd.grad(y, leaf, torch.ones_like(y))
