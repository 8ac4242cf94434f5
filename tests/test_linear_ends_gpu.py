"""odie_amd.linear at the ends of its types: sums past fp16's range, and infinite sums.  Inputs are powers of two and
small whole numbers, so that every sum is exact in each type; at the large ones an activation and its slope are at
their limits."""
import pytest
import torch

from odie_amd.linear import ACTIVATIONS, linear
from rows64 import DTYPES, Layer64, check

pytestmark = pytest.mark.gpu

# value and slope for sums far below and far above 0, as (constant, multiple of the sum)
BELOW = {'none': ((0, 1), 1), 'relu': ((0, 0), 0), 'sigmoid': ((0, 0), 0), 'softplus': ((0, 0), 0), 'gelu': ((0, 0), 0),
         'silu': ((0, 0), 0)}
ABOVE = {'none': ((0, 1), 1), 'relu': ((0, 1), 1), 'sigmoid': ((1, 0), 0), 'softplus': ((0, 1), 1), 'gelu': ((0, 1), 1),
         'silu': ((0, 1), 1)}


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('activation', ACTIVATIONS)
@pytest.mark.parametrize('n', (6, 200))       # weights read straight into registers, and by tiles
def test_sums_past_the_range_of_fp16(n, activation, dtype):
    """Column 0 sums to -131072 or 131072, which fp16 does not hold; column 1 to small numbers, alone."""
    print('linear', n, activation, dtype, flush=True)
    sign = torch.where(torch.arange(n, device='cuda') % 3 == 0, 1.0, -1.0)
    small = (torch.arange(n, device='cuda') % 5 - 2).float()
    x = torch.zeros(n, 8, device='cuda')
    x[:, 0], x[:, 1] = 256 * sign, small
    w = torch.zeros(2, 8, device='cuda')
    w[0, 0], w[1, 1] = 512, 1
    dy = torch.zeros(n, 2, device='cuda')
    dy[:6] = torch.tensor([[1, 1], [-1, 2], [2, -1], [1, 1], [2, 1], [-1, -2]], device='cuda')
    x, w, dy = x.to(dtype).requires_grad_(True), w.to(dtype).requires_grad_(True), dy.to(dtype)
    b = torch.zeros(2, dtype=dtype, device='cuda', requires_grad=True)
    y = linear(x, w, b, activation=activation)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    z = 131072 * sign
    below, above = BELOW[activation], ABOVE[activation]
    value = torch.where(z < 0, below[0][0] + below[0][1] * z, above[0][0] + above[0][1] * z)
    dz = dy[:, 0].float() * torch.where(z < 0, float(below[1]), float(above[1]))
    assert torch.equal(y[:, 0].detach(), value.to(dtype))
    assert torch.equal(dx[:, 0].float(), 512 * dz) and not dx[:, 2:].any()
    assert torch.equal(dw[0, :2].float(), torch.stack(((dz * 256 * sign).sum(), (dz * small).sum()))) and not dw[:, 2:].any()
    assert db[0].float() == dz.sum()
    other = Layer64(x[:, 1:2], w[1:, 1:2], b[1:], None, dy[:, 1:], activation)
    check(y[:, 1:], other.y, other.y_error, 'y')
    if activation != 'relu':        # its slope jumps at 0, which column 1 holds
        check(dx[:, 1:2], other.dx, other.dx_error, 'dx')
        check(db[1:], other.db, other.db_error, 'db')
        check(dw[1:, 1:2], other.dw, other.dw_error, 'dw')


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('activation', ACTIVATIONS)
def test_slopes_of_infinite_sums(activation, dtype):
    """Slopes at infinity are their limits, and the value is where it is one."""
    infinity = float('inf')
    x = torch.tensor([[-infinity], [infinity]], device='cuda', dtype=dtype).requires_grad_(True)
    y = linear(x, torch.ones(1, 1, device='cuda', dtype=dtype), activation=activation)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert dx.flatten().tolist() == [BELOW[activation][1], ABOVE[activation][1]]
    assert y[1].item() == (1 if activation == 'sigmoid' else infinity)
    if activation in ('relu', 'sigmoid', 'softplus'):
        assert y[0].item() == 0
