"""examples/blended_experts.py: the row operators in one training program."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parent.parent / 'examples' / 'blended_experts.py'
    spec = importlib.util.spec_from_file_location('blended_experts', path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_weights_blend_the_surrounding_tiles():
    """Bilinear weights over tile centres reproduce the position itself (away from the outer border), and sum to 1."""
    module = _example()
    coords = torch.rand(1000, 2, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda')
    expert, weights = module.surrounding_tiles(coords, 5, 4)
    assert ((expert >= -1) & (expert < 20)).all() and (weights[expert < 0] == 0).all()
    assert (weights.sum(1) - 1).abs().max() < 1e-6
    centres = torch.stack(((expert % 5 + 0.5) / 5, (torch.div(expert, 5, rounding_mode='floor') + 0.5) / 4), 2)
    inner = (expert >= 0).all(1)
    assert inner.any() and ((centres * weights[..., None]).sum(1) - coords)[inner].abs().max() < 1e-5


def test_the_fit_learns():
    """The error of a fit falls below half of where it starts within 60 steps, and the same run gives the same bits."""
    module = _example()
    first = module.main(steps=60, height=96, width=128, regions_x=4, regions_y=3, batch=4096)
    assert first.isfinite().all() and first[-5:].mean() < 0.5 * first[:5].mean()
    assert torch.equal(module.main(steps=60, height=96, width=128, regions_x=4, regions_y=3, batch=4096), first)
