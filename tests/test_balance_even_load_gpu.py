"""odie_amd.router.balance where the load is nearly even, as its loss makes it: the gradient is of the counts' differences
from their mean under a row's softmax, which are far smaller than the counts.

With p off by `off` relative, the whole numbers c - M / E are exact, and a sum over E of them has the bound of an fp32 sum
of their magnitudes: nothing is relative to the counts themselves."""
import pytest
import torch

from odie_amd.router import balance
from rows64 import DTYPES, check, rounding
from test_router_gpu import FAINT, _softmax64

pytestmark = pytest.mark.gpu


# rows of some lanes (counts past 2^24 too), of a wave, of a workgroup, and longer ones
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n, width, each', ((4096, 2, (1 << 25) + 1), (4096, 8, 1000000), (512, 1000, 16000), (256, 5000, 3000),
                                            (64, 10000, 900), (64, 20000, 900)))
def test_gradient_of_a_nearly_even_load(n, width, each, dtype):
    print('even load', n, width, each, dtype, flush=True)
    generator = torch.Generator(device='cuda').manual_seed(width)
    counts = torch.randint(-3, 4, (width,), generator=generator, device='cuda') + each
    entries = int(counts.sum())
    choices = (entries + n - 1) // n
    expert = torch.full((n * choices,), -1, dtype=torch.int32, device='cuda')
    expert[:entries] = torch.repeat_interleave(torch.arange(width, dtype=torch.int32, device='cuda'), counts)
    # every row has entries of several experts and of none
    expert = expert.view(choices, n).t().contiguous()
    logits = (torch.randn(n, width, generator=generator, device='cuda') * 2).to(dtype)
    leaf = logits.clone().requires_grad_(True)
    loss, got = balance(leaf, expert)
    scale = float(n)
    gradient, = torch.autograd.grad(loss, leaf, torch.tensor(scale, device='cuda'))
    assert torch.equal(got.long(), counts)

    p, off, _ = _softmax64(logits)
    norm = width / (entries * n)
    apart = (counts - round(entries / width)).double()          # exact
    t = (p * apart).sum(1, keepdim=True)
    size = (p * apart.abs()).sum(1, keepdim=True)
    t_off = (p * apart.abs() * (off + 2.0 ** -23)).sum(1, keepdim=True) + 1.1 * (2 * width + 6) * 2.0 ** -24 * size
    expected = norm * (t.sum() + n * float(round(entries / width)))
    check(loss, expected, norm * t_off.sum() + 2.0 ** -23 * expected, 'loss')
    d = scale * norm * p * (apart - t)
    d_off = scale * norm * (p * (off + 2.0 ** -21) * (apart - t).abs() + p * (t_off + 2.0 ** -23 * (apart.abs() + t.abs()))) + FAINT
    check(gradient, d, d_off * 1.01 + rounding(dtype, d), 'gradient')
