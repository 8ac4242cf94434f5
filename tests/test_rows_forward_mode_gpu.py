"""Forward-mode derivatives, which the row operators do not have, are refused and not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from odie_amd.embedding import embed
from odie_amd.linear import linear
from odie_amd.mixture import combine, dispatch, expert_order

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    x, w, b, r = (torch.ones(*shape, device='cuda') for shape in ((4, 8), (6, 8), (6,), (4, 6)))
    order = expert_order(torch.arange(4, device='cuda'), 4)
    ids = torch.zeros(3, dtype=torch.int64, device='cuda')
    weights = torch.ones(4, 1, device='cuda')
    calls = [(x, lambda t: linear(t, w)), (w, lambda t: linear(x, t)), (b, lambda t: linear(x, w, t)),
             (r, lambda t: linear(x, w, residual=t)), (x, lambda t: dispatch(t, order)), (x, lambda t: combine(t, order)),
             (weights, lambda t: combine(x, order, t)), (weights.half(), lambda t: combine(x, order, t)),
             (x, lambda t: embed(t, ids))]
    for value, call in calls:
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(value, torch.ones_like(value))
            with pytest.raises(NotImplementedError):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError):   # which leaves forward mode on
                call(dual)
            assert torch.equal(call(value), call(value.clone()))        # without a tangent, as ever
