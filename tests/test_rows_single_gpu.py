"""The row operators on one row or one column whose strides torch leaves as they were: a transposed column, an expanded
upstream."""
import pytest
import torch

from odie_amd.embedding import embed
from odie_amd.linear import linear
from odie_amd.mixture import combine, dispatch, expert_order
from rows64 import DTYPES

pytestmark = pytest.mark.gpu


def _row(generator, width, dtype):
    """[1, width] with strides (1, 1), and the same values with strides (width, 1)."""
    column = torch.randn(width, 1, generator=generator, device='cuda').to(dtype)
    row = column.t()
    assert row.stride() == (1, 1) and row.is_contiguous()
    return row, column.flatten().clone().view(1, width).as_strided((1, width), (width, 1))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_linear_of_a_transposed_column(dtype):
    generator = torch.Generator(device='cuda').manual_seed(1)
    w = torch.randn(24, 64, generator=generator, device='cuda').to(dtype).requires_grad_(True)
    (x, dense_x), (r, dense_r), (dy, dense_dy) = (_row(generator, width, dtype) for width in (64, 24, 24))
    got, expected = [], []
    for into, a, b, up in ((got, x, r, dy), (expected, dense_x, dense_r, dense_dy)):
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        y = linear(a, w, activation='silu', residual=b)
        into.extend((y.detach(), *torch.autograd.grad(y, (a, w, b), up)))
    assert all(torch.equal(a, b) for a, b in zip(got, expected))
    # the upstream of a transposed result has strides (1, 1)
    y = linear(dense_x, w, activation='silu')
    dw, = torch.autograd.grad(y.t(), w, dense_dy.t().contiguous())
    again, = torch.autograd.grad(linear(dense_x, w, activation='silu'), w, dense_dy)
    assert torch.equal(dw, again)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_exchange_and_lookup_of_a_transposed_column(dtype):
    generator = torch.Generator(device='cuda').manual_seed(2)
    row, dense = _row(generator, 40, dtype)
    order = expert_order(torch.tensor([[2]], device='cuda'), 4)
    ids = torch.zeros(1, dtype=torch.int64, device='cuda')
    weights = torch.full((1, 1), 0.5, device='cuda', requires_grad=True)
    for call in (lambda t: dispatch(t, order), lambda t: combine(t, order), lambda t: combine(t, order, weights),
                 lambda t: embed(t, ids, 2.0)):
        got, expected = [], []
        for into, t in ((got, row), (expected, dense)):
            t = t.detach().requires_grad_(True)
            y = call(t)
            into.extend((y.detach(), *torch.autograd.grad(y.t(), t, dense.t().contiguous())))
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_sums_of_one_value(dtype):
    """The gradient of a sum arrives expanded, with strides (0, 0), which torch calls contiguous for one value."""
    one = torch.ones(1, 1, dtype=dtype, device='cuda')
    order = expert_order(torch.tensor([[0]], device='cuda'), 1)
    ids = torch.zeros(1, dtype=torch.int64, device='cuda')
    weights = torch.full((1, 1), 3.0, device='cuda')
    for call, slope in ((lambda t: linear(t, 3 * one), 3), (lambda t: linear(one, t, activation='silu'), None),
                        (lambda t: dispatch(t, order), 1), (lambda t: combine(t, order, weights), 3),
                        (lambda t: embed(t, ids, 3.0), 3)):
        t = (2 * one).requires_grad_(True)
        got, = torch.autograd.grad(call(t).sum(), t)
        other, = torch.autograd.grad(call(t), t, one)
        assert torch.equal(got, other) and (slope is None or got.item() == slope)


@pytest.mark.parametrize('n', (1, 2, 70))
def test_one_column_of_any_stride(n):
    generator = torch.Generator(device='cuda').manual_seed(3)
    wide = torch.randn(n, 6, generator=generator, device='cuda')
    w = torch.randn(5, 1, generator=generator, device='cuda')
    order = expert_order(torch.arange(n, device='cuda') % 3, 3)
    dense = wide[:, 2:3].clone()
    for column in (wide[:, 2:3], wide[:, 2::3][:, :1], wide.t().contiguous().t()[:, 2:3], dense.as_strided((n, 1), (1, 0))):
        assert torch.equal(column, dense)
        assert torch.equal(linear(column, w), linear(dense, w))
        assert torch.equal(dispatch(column, order), dispatch(dense, order))
    same = dense[:1].expand(n, 1)
    assert torch.equal(linear(same, w), linear(same.clone(), w))
