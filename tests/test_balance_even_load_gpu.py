"""odie_amd.router.balance where a row's mean count is far larger than the counts' differences from it, of which the gradient
is: in a load that is nearly even, as its loss makes it, and in rows that are sure of one expert.

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


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n, width', ((4096, 8), (4096, 64), (512, 1000), (256, 5000), (64, 10000), (64, 20000)))
def test_gradient_of_an_uneven_load(n, width, dtype):
    """Counts from 1 to 2^17 and rows that are sure of one expert, rare or popular: a row's differences are from its own mean
    count, far smaller than that count and than M / E.

    A whole number within 1.5 of a row's mean comes off the counts exactly (half a unit by its rounding, and the first
    sum's error: 2^17 times 2^-24 times the roundings of about 30 terms a lane and 8 steps between lanes is below 1), so
    that only what is left, |c - t| + 1.5 each, is rounded.  Rows that a lane does not hold (more than 8192 fp32 and 16384
    16-bit logits) have M / E or nothing taken off: relative to t, or to t + M / E where t is above a third of that."""
    print('uneven load', n, width, dtype, flush=True)
    generator = torch.Generator(device='cuda').manual_seed(width)
    counts = 1 + (torch.arange(width, device='cuda') * 7 % 18 == torch.arange(width, device='cuda') % 18).long()
    counts = counts + (1 << (torch.arange(width, device='cuda') * 5 % 18)) * (torch.arange(width, device='cuda') < 400)
    entries = int(counts.sum())
    choices = (entries + n - 1) // n
    expert = torch.full((n * choices,), -1, dtype=torch.int32, device='cuda')
    expert[:entries] = torch.repeat_interleave(torch.arange(width, dtype=torch.int32, device='cuda'), counts)
    expert = expert.view(choices, n).t().contiguous()
    assert (expert >= 0).any(1).all()
    logits = torch.randn(n, width, generator=generator, device='cuda')
    sure = torch.randint(0, min(width, 400), (n,), generator=generator, device='cuda')
    logits[torch.arange(n, device='cuda'), sure] = 14.0 + 4 * torch.rand(n, generator=generator, device='cuda')
    logits = logits.to(dtype)
    leaf = logits.clone().requires_grad_(True)
    loss, got = balance(leaf, expert)
    scale = float(n)
    gradient, = torch.autograd.grad(loss, leaf, torch.tensor(scale, device='cuda'))
    assert torch.equal(got.long(), counts)

    p, off, _ = _softmax64(logits)
    norm = width / (entries * n)
    c = counts.double()
    t = (p * c).sum(1, keepdim=True)
    apart = c - t
    size = apart.abs() + 1.5
    if width > (8192 if dtype == torch.float32 else 16384):
        mean = entries / width
        size = c + t + torch.where(t > mean / 3, mean, 0.0)
    total = (p * size).sum(1, keepdim=True)
    t_off = (p * size * (off + 2.0 ** -23)).sum(1, keepdim=True) + 1.1 * (2 * width + 6) * 2.0 ** -24 * total
    expected = norm * t.sum()
    check(loss, expected, norm * t_off.sum() + 2.0 ** -23 * expected, 'loss')
    d = scale * norm * p * apart
    d_off = scale * norm * (p * (off + 2.0 ** -21) * apart.abs() + p * (t_off + 2.0 ** -23 * (size + 1.5))) + FAINT
    check(gradient, d, d_off * 1.01 + rounding(dtype, d), 'gradient')
