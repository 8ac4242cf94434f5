"""The router's operators and quantisation past 2^31 elements and 2^32 bytes: rows far into large tensors are read and written
where they lie."""
import pytest
import torch

from odie_amd.linear import linear
from odie_amd.microscale import quantize
from odie_amd.router import balance, choose, distill

pytestmark = pytest.mark.gpu

WIDTH = 32760
ROWS = (1 << 31) // WIDTH + 99     # 2.15e9 bf16 values, 4.3 GB


def _logits(rows, width):
    """Rows that differ: a pattern along the columns, moved on by each row."""
    value = torch.empty(rows, width, dtype=torch.bfloat16, device='cuda')
    column = torch.arange(width, device='cuda')
    for at in range(0, rows, 4096):
        row = torch.arange(at, min(rows, at + 4096), device='cuda')[:, None]
        value[at:at + 4096] = ((column * 37 + row * 101) % 1009).to(torch.bfloat16) / 128
    return value


@pytest.fixture(scope='module')
def logits():
    return _logits(ROWS, WIDTH)


PARTS = (slice(0, 3), slice((1 << 31) // WIDTH - 2, (1 << 31) // WIDTH + 3), slice(ROWS - 3, ROWS))


@pytest.mark.parametrize('normalize', (True, False))
def test_choices(logits, normalize):
    print('choose', tuple(logits.shape), flush=True)
    leaf = logits.detach().requires_grad_(True)
    expert, weights = choose(leaf, 3, normalize=normalize)
    upstream = torch.ones_like(weights)
    upstream[:, 1] = -2
    gradient, = torch.autograd.grad(weights, leaf, upstream)
    for part in PARTS:
        some = logits[part].clone().requires_grad_(True)
        e, w = choose(some, 3, normalize=normalize)
        assert torch.equal(expert[part], e) and torch.equal(weights[part], w)
        assert torch.equal(gradient[part], torch.autograd.grad(w, some, upstream[part])[0])


def test_balance(logits):
    """The rows before the last ones take no part: the loss and the gradient are the last rows' own."""
    print('balance', tuple(logits.shape), flush=True)
    expert = torch.full((ROWS, 2), -1, dtype=torch.int32, device='cuda')
    expert[-5:] = torch.arange(10, device='cuda', dtype=torch.int32).view(5, 2) * 3000
    leaf = logits.detach().requires_grad_(True)
    loss, counts = balance(leaf, expert)
    gradient, = torch.autograd.grad(loss, leaf)
    some = logits[-5:].clone().requires_grad_(True)
    own, own_counts = balance(some, expert[-5:])
    assert torch.equal(counts, own_counts) and torch.equal(loss, own)
    assert torch.equal(gradient[-5:], torch.autograd.grad(own, some)[0]) and not gradient[:-5].any()


def test_distillation(logits):
    print('distill', tuple(logits.shape), flush=True)
    ids = (torch.arange(ROWS * 4, device='cuda').view(ROWS, 4) * 7919) % WIDTH
    teacher = (torch.arange(ROWS * 4, device='cuda').view(ROWS, 4) % 5).float()
    leaf = logits.detach().requires_grad_(True)
    loss = distill(leaf, ids, teacher)
    gradient, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    for part in PARTS:
        some = logits[part].clone().requires_grad_(True)
        own = distill(some, ids[part], teacher[part])
        # few rows are cut into pieces, whose sums are joined in another order: 2^-20 of a loss of about ten
        assert (loss[part] - own).abs().max() < 2.0 ** -16
        expected, = torch.autograd.grad(own, some, torch.ones_like(own))
        assert (gradient[part].double() - expected.double()).abs().max() <= 2.0 ** -7 * float(expected.abs().max())


def test_quantisation_and_product(logits):
    print('quantize', tuple(logits.shape), flush=True)
    q = quantize(logits)
    back = q.dequantize()
    weight = quantize(_logits(40, WIDTH))
    y, y4 = linear(logits, weight), linear(q, weight)
    for part in PARTS:
        own = quantize(logits[part])
        assert torch.equal(q.codes[part], own.codes) and torch.equal(q.scales[part], own.scales)
        assert torch.equal(back[part], own.dequantize())
        # few rows split the depth over waves: fp32 sums of 32760 products in another order, and one rounding to bf16
        for full, few in ((y[part], linear(logits[part], weight)), (y4[part], linear(own, weight))):
            assert (full.double() - few.double()).abs().max() <= 2.0 ** -7 * float(few.abs().max())
