"""Arguments of the row operators that are no tensors are refused like those of wrong shapes."""
import pytest
import torch

from odie_amd.linear import linear
from odie_amd.mixture import combine, dispatch, expert_order

pytestmark = pytest.mark.gpu


def test_arguments_that_are_no_tensors():
    x, w = torch.zeros(4, 8, device='cuda'), torch.zeros(2, 6, 8, device='cuda')
    order = expert_order(torch.zeros(4, 1, dtype=torch.int32, device='cuda'), 3)
    for bad in (lambda: linear(x, w[0], [0.0] * 6), lambda: linear(x, w[0], 1.0), lambda: linear(x, w, offsets=[0, 2, 4]),
                lambda: linear(x, w[0], residual=0.0), lambda: linear(x.tolist(), w[0]), lambda: linear(x, w[0].tolist()),
                lambda: combine(x, order, [[1.0]] * 4), lambda: combine(x, order, 1.0), lambda: combine(x.tolist(), order),
                lambda: dispatch(x.tolist(), order), lambda: expert_order([0, 1], 3),
                lambda: expert_order(order.slots, 2.5), lambda: expert_order(order.slots, None)):
        with pytest.raises(ValueError):
            bad()
