"""gelu's left tail, to its own magnitude."""
import math

import pytest
import torch

from odie_amd.linear import linear
from rows64 import DTYPES, TINY, UNIT, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n', (64, 4096))
def test_the_left_tail_of_gelu(n, dtype):
    """z Phi(z) for z down to -14 to its own magnitude.  Beside the last rounding: exp(-z^2 / 2) from an exponent of at
    most 142 with three roundings (142 x 3 x 2^-24 ln 2 < 2^-15), erfc's other factor (2^-20), a few products (2^-20);
    in all below 2^-14.  exp(-z^2 / 2) below 2^-126 may count as 0."""
    z = torch.linspace(-14, 0, n, device='cuda').to(dtype)
    x = torch.zeros(n, 8, dtype=dtype, device='cuda')
    x[:, 0] = z
    w = torch.zeros(8, 8, dtype=dtype, device='cuda')
    w[:, 0] = 1
    y = linear(x, w, activation='gelu')
    expected = (z.double() * 0.5 * torch.erfc(-z.double() * math.sqrt(0.5)))[:, None].expand(n, 8)
    check(y, expected, (UNIT[dtype] * 1.001 + 2.0 ** -14) * expected.abs() + TINY[dtype] + 14 * 2.0 ** -126, 'gelu')
