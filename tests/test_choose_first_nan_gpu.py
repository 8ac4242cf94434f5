"""odie_amd.router.choose where the first expert's logit is a NaN: the largest of its row whatever the row's length, the
number of rows and the choices are."""
import math

import pytest
import torch

from odie_amd.router import choose
from rows64 import DTYPES

pytestmark = pytest.mark.gpu


# rows of some lanes, of a wave, of a workgroup, and of fp32 that are read once a choice: by their length, or by their
# number and few choices
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('normalize', (True, False))
@pytest.mark.parametrize('n, width, choices', ((8, 5, 3), (8, 300, 3), (8, 2100, 1), (1030, 2100, 1), (1030, 5000, 4), (8, 20000, 3),
                                               (8, 32768, 4)))
def test_the_first_of_a_row(n, width, choices, normalize, dtype):
    print('choose', n, width, choices, dtype, normalize, flush=True)
    generator = torch.Generator(device='cuda').manual_seed(width)
    logits = torch.randn(n, width, generator=generator, device='cuda').to(dtype)
    logits[1, 0], logits[2, 0] = math.nan, -math.nan
    logits[3] = -math.inf
    logits[3, 0] = math.nan
    logits[4, 0], logits[4, 3] = math.nan, math.inf
    logits[5, 0], logits[5, 4] = math.nan, math.nan
    clean = torch.cat((logits[:1], logits[6:]))
    leaf = logits.requires_grad_(True)
    expert, weights = choose(leaf, choices, normalize=normalize)
    assert (expert[1:6, 0] == 0).all() and weights[1:6, 0].isnan().all()
    assert (expert[3, 1:] == -1).all() and not weights[3, 1:].any()
    if choices > 1:
        assert expert[4, 1] == 3 and expert[5, 1] == 4
        held = torch.tensor([1, 2, 4, 5], device='cuda')
        assert weights[held].isnan().all()
    others = torch.cat((expert[:1], expert[6:])), torch.cat((weights[:1], weights[6:]))
    alone = choose(clean.detach(), choices, normalize=normalize)
    assert torch.equal(others[0], alone[0])
    assert torch.allclose(others[1], alone[1], rtol=2.0 ** -18, atol=0.0)     # few and many rows may go different ways
    gradient, = torch.autograd.grad(weights.sum(), leaf)
    assert gradient[1:6, 0].isnan().all()
    assert not gradient[0].isnan().any() and not gradient[6:].isnan().any()
