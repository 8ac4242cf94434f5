"""RoutedMixture's experts chosen by fp32 logits beside 16-bit layers, as its docstring writes it."""
import pytest
import torch

from odie_amd.linear import linear
from odie_amd.mixture import RoutedMixture
from odie_amd.router import balance, choose

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', (torch.float16, torch.bfloat16), ids=str)
def test_choice_by_fp32_logits(dtype):
    torch.manual_seed(1)
    m = RoutedMixture(16, 2, 32, 64, 5, dtype=dtype, seed=4)
    x = torch.randn(3000, 32, device='cuda', dtype=dtype, requires_grad=True)
    logits = linear(x.float(), m.router.float())
    expert, weights = choose(logits, m.choices)
    y = m.mixture(x, expert, weights)
    # sums of 32 exact products in fp32: choices whose logits lie further apart are the exact ones
    exact = x.detach().double() @ m.router.detach().double().t()
    off = 34 * 2.0 ** -23 * (x.detach().double().abs() @ m.router.detach().double().abs().t()).amax(1)
    top = exact.topk(3, dim=1)
    clear = ((top.values[:, :2] - top.values[:, 1:]) > 2 * off[:, None]).all(1)
    assert clear.float().mean() > 0.99
    assert torch.equal(expert[clear].long(), top.indices[clear, :2])
    # rounded logits tie or change places in some of these rows
    assert not torch.equal(m(x)[2][clear].long(), top.indices[clear, :2])
    loss = y.float().square().mean() + 0.1 * balance(logits, expert)[0]
    grads = torch.autograd.grad(loss, [x, m.router, *m.mixture.parameters()])
    assert grads[0].dtype == grads[1].dtype == dtype
    assert all(g.isfinite().all() and g.any() for g in grads)
