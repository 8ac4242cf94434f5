"""odie_amd.microscale.quantize has no forward-mode derivative: a tangent is refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from odie_amd.microscale import quantize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('shape', ((4, 64), (2, 3, 40)), ids=str)
def test_tangents_are_refused(shape):
    x = torch.randn(*shape, device='cuda')
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError):
                quantize(dual)
            assert torch.equal(quantize(x).codes, quantize(x.clone()).codes)        # without a tangent, as ever
