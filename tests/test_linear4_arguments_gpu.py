"""odie_amd.linear with rows of 4 bits refuses a bias or residual that is no tensor with the errors of the other layers."""
import pytest
import torch

from odie_amd.linear import linear
from odie_amd.microscale import quantize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('value', (3.0, [0.0] * 6, 'bias'), ids=str)
def test_bias_and_residual_that_are_no_tensors(value):
    x, w = torch.randn(4, 64, device='cuda'), quantize(torch.randn(6, 64, device='cuda'))
    for rows in (x, quantize(x)):
        with pytest.raises(ValueError, match='bias'):
            linear(rows, w, value)
        with pytest.raises(ValueError, match='residual'):
            linear(rows, w, residual=value)
