"""odie_amd.router.balance of an empty batch, however many experts there are."""
import pytest
import torch

from odie_amd.router import balance
from rows64 import DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', (1, 64, 9000, 16384, 16385, 32768))
def test_no_rows_of_many_experts(width, dtype):
    for choices in (1, 5):
        x = torch.zeros(0, width, device='cuda', dtype=dtype, requires_grad=True)
        expert = torch.zeros(0, choices, device='cuda', dtype=torch.int32)
        loss, counts = balance(x, expert)
        assert loss == 0 and counts.shape == (width,) and not counts.any()
        assert torch.autograd.grad(loss, x)[0].shape == (0, width)
        assert balance(x.detach(), expert)[0] == 0
