"""The row operators past 2^32 bytes and 2^31 elements: rows far into large tensors are read and written where they lie."""
import pytest
import torch

from odie_amd.embedding import embed
from odie_amd.linear import linear
from odie_amd.mixture import combine, dispatch, expert_order

pytestmark = pytest.mark.gpu

WIDTH = 1032
ROWS = (1 << 21) + 77          # of WIDTH fp16 values: 2.16e9 elements, 4.3 GB


def _filled(rows, width, dtype=torch.float16):
    """Row i holds the whole number i % 97 + (column % 5), exact in fp16."""
    value = torch.empty(rows, width, dtype=dtype, device='cuda')
    value.copy_((torch.arange(rows, device='cuda') % 97).to(dtype)[:, None])
    value += (torch.arange(width, device='cuda') % 5).to(dtype)
    return value


def test_lookup_in_a_large_table():
    print('lookup', ROWS, WIDTH, flush=True)
    table = _filled(ROWS, WIDTH).requires_grad_(True)
    ids = torch.tensor([0, ROWS - 1, ROWS - 2, ROWS // 2, ROWS - 1, (1 << 31) // WIDTH + 1], device='cuda')
    y = embed(table, ids, 2.0)
    assert torch.equal(y, table.detach()[ids] * 2)
    dtable, = torch.autograd.grad(y, table, torch.ones_like(y))
    assert (dtable[ROWS - 1] == 4).all() and (dtable[ROWS // 2] == 2).all() and (dtable[1] == 0).all()
    assert int(dtable.count_nonzero()) == 5 * WIDTH


def test_exchange_of_many_rows():
    n = ROWS
    print('exchange', n, WIDTH, flush=True)
    x = _filled(n, WIDTH)
    expert = torch.arange(n, device='cuda') % 3
    order = expert_order(expert, 3)
    sent = dispatch(x, order)
    assert torch.equal(sent[-5:], x[order.source[-5:].long()]) and torch.equal(sent[:5], x[0:15:3])
    back = combine(sent, order)
    assert torch.equal(back[-1000:], x[-1000:]) and torch.equal(back[(1 << 31) // WIDTH - 3:][:9], x[(1 << 31) // WIDTH - 3:][:9])
    del sent
    weights = torch.full((n, 1), 0.5, device='cuda', requires_grad=True)
    rows = x.requires_grad_(True)
    y = combine(rows, order, weights)
    drows, dweights = torch.autograd.grad(y, (rows, weights), torch.ones_like(y))
    assert (drows[-1000:] == 0.5).all()
    last = order.slots[-1000:, 0].long()
    assert torch.equal(dweights[-1000:, 0], rows.detach()[last].double().sum(1).float())


def test_linear_over_many_rows():
    """Inputs and outputs of a layer past 2^31 elements, whole numbers throughout: the last rows exact."""
    n, inputs, outputs = ROWS, WIDTH, 1088
    print('linear', n, inputs, outputs, flush=True)
    x = torch.zeros(n, inputs, dtype=torch.float16, device='cuda')
    x[-300:] = _filled(300, inputs)
    x.requires_grad_(True)
    weight = torch.zeros(outputs, inputs, dtype=torch.float16, device='cuda')
    weight[torch.arange(outputs), torch.arange(outputs) % inputs] = 2
    weight.requires_grad_(True)
    y = linear(x, weight)
    expected = 2 * x.detach()[-300:][:, torch.arange(outputs, device='cuda') % inputs]
    assert torch.equal(y.detach()[-300:], expected) and not y.detach()[:-300].any()
    up = torch.zeros_like(y)
    up[-300:] = 1
    dx, dw = torch.autograd.grad(y, (x, weight), up)
    times = torch.bincount(torch.arange(outputs, device='cuda') % inputs, minlength=inputs).half() * 2
    assert torch.equal(dx[-300:], times.expand(300, inputs)) and not dx[:-300].any()
    assert torch.equal(dw, x.detach()[-300:].double().sum(0).half().expand(outputs, inputs))
