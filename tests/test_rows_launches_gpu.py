"""Calls of more workgroups than one launch takes (2^32 threads): the rows past the first launch's are done too."""
import pytest
import torch

from odie_amd.linear import linear
from odie_amd.mixture import combine, dispatch, expert_order

pytestmark = pytest.mark.gpu


def test_exchange_of_more_rows_than_a_launch():
    """67 million rows of 257 values, 64 lanes each."""
    n, width = (1 << 26) + 1029, 257
    print('exchange', n, width, flush=True)
    x = torch.empty(n, width, dtype=torch.float16, device='cuda')
    x.copy_((torch.arange(n, device='cuda') % 97).half()[:, None])
    x += (torch.arange(width, device='cuda') % 5).half()
    expert = (torch.arange(n, device='cuda') % 7).to(torch.int32)
    expert[-3] = -1
    order = expert_order(expert, 7)
    del expert
    sent = dispatch(x, order)
    for begin in range(0, n - 1, 1 << 23):                 # the last place is the lost row's
        part = slice(begin, min(begin + (1 << 23), n - 1))
        assert torch.equal(sent[part], x[order.source[part].long()]), begin
    assert not sent[-1].any()
    weights = torch.ones(n, 1, device='cuda', requires_grad=True)
    sent.requires_grad_(True)
    y = combine(sent, order, weights)
    squares = torch.empty(n, device='cuda')
    for begin in range(0, n, 1 << 23):
        part = slice(begin, min(begin + (1 << 23), n))
        squares[part] = x[part].float().square().sum(1)     # whole numbers below 2^24
    squares[-3] = 0
    x[-3] = 0
    assert torch.equal(y.detach(), x)
    del x
    drows, dweights = torch.autograd.grad(y, (sent, weights), y.detach())
    assert torch.equal(drows, sent.detach()) and torch.equal(dweights[:, 0], squares)


def test_linear_over_more_rows_than_a_launch():
    """A thousand million rows of one value each, whole numbers: the last ones exact."""
    n = (1 << 30) + 1000
    print('linear', n, flush=True)
    x = torch.zeros(n, 1, dtype=torch.float16, device='cuda')
    x[::65536] = 1
    x[-2000:] = (torch.arange(2000, device='cuda') % 11).half()[:, None]
    x.requires_grad_(True)
    w = torch.full((2, 1), 3.0, dtype=torch.float16, device='cuda')
    w[1] = -1
    y = linear(x, w)
    assert torch.equal(y.detach()[:, 0], 3 * x.detach()[:, 0]) and torch.equal(y.detach()[:, 1], -x.detach()[:, 0])
    dx, = torch.autograd.grad(y, x, y.detach())
    assert torch.equal(dx, 10 * x.detach())
