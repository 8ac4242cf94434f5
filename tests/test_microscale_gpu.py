"""odie_amd.microscale: codes and scales bit for bit against 64-bit arithmetic, and back."""
import math

import pytest
import torch

from microscale64 import quantize64, values64
from odie_amd.microscale import Microscaled, quantize
from rows64 import DTYPES

pytestmark = pytest.mark.gpu

SHAPES = ((1, 1), (3, 7), (2, 31), (5, 32), (4, 33), (7, 64), (9, 127), (70, 128), (33, 129), (6, 1000), (3, 2048), (2, 8191),
          (1000, 40), (300, 2056))


def _check(x, what):
    q = quantize(x)
    flat = x.reshape(-1, x.shape[-1])
    codes, scales = quantize64(flat)
    assert q.shape == x.shape and q.dtype == x.dtype and q.ndim == x.ndim and q.device == x.device
    got = q.codes.reshape(codes.shape).cpu(), q.scales.reshape(scales.shape).cpu()
    assert torch.equal(got[1], scales), what
    # a NaN block's codes are 0; else -0 is told from 0
    assert torch.equal(got[0], codes), what
    for dtype in DTYPES:
        back = q.dequantize(dtype)
        expected = values64(codes, scales, x.shape[-1]).to(dtype).view(x.shape)
        assert back.dtype == dtype and torch.equal(back.cpu().isnan(), expected.isnan()), what
        assert torch.equal(back.cpu().nan_to_num(7.0), expected.nan_to_num(7.0)), (what, dtype)
    assert torch.equal(q.dequantize().nan_to_num(7.0), q.dequantize(x.dtype).nan_to_num(7.0))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_quantize_and_back(shape, dtype):
    print('quantize', shape, dtype, flush=True)
    generator = torch.Generator(device='cuda').manual_seed(shape[0] + shape[1])
    size = torch.exp(2 * torch.randn(1, shape[1], generator=generator, device='cuda'))
    _check((torch.randn(*shape, generator=generator, device='cuda') * size).to(dtype), str(shape))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_every_border(dtype):
    """Each middle between two codes, its neighbours of the type, and both signs, at small, usual and large scales."""
    borders = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0])
    least = -20 if dtype == torch.float16 else -120
    for power in (least, -3, 0, 11):
        v = (borders * 2.0 ** power).to(dtype)
        step = torch.finfo(dtype).eps
        for near in (v, (v.double() * (1 + step)).to(dtype), (v.double() * (1 - step)).to(dtype)):
            row = torch.cat((near, -near)).view(1, 32)
            row[0, 14] = 4 * 2.0 ** power      # the largest of 7 or 4 to 8: the scale is this power of two
            _check(row.cuda(), (power, dtype))
            row[0, 15] = row[0, 31] = 0
            _check(row.cuda(), (power, dtype))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_ends_of_the_range(dtype):
    """Blocks of zeros, of -0, of the least and largest values; of NaN and infinities, whose neighbours stay as they are."""
    info = torch.finfo(dtype)
    x = torch.zeros(6, 96, device='cuda', dtype=dtype)
    x[1] = -0.0
    x[2, ::3] = info.smallest_normal
    x[2, 40] = info.smallest_normal / 4
    x[3] = info.smallest_normal * info.eps      # the least subnormal
    x[3, 5] *= 3
    x[4], x[4, 64] = info.max, info.min
    x[5] = 1.0
    x[5, 3], x[5, 95] = math.nan, -math.inf
    _check(x, 'ends')
    back = quantize(x).dequantize()
    assert back[5, :32].isnan().all() and back[5, 64:].isnan().all() and (back[5, 32:64] == 1).all()


def test_strides_and_dimensions():
    generator = torch.Generator(device='cuda').manual_seed(2)
    wide = torch.randn(40, 150, generator=generator, device='cuda')
    for x in (wide[:, 3:104], wide[::2, 1:66], wide.t(), wide[5:6, 7:90], wide.view(4, 10, 150), wide.view(4, 10, 150)[:, ::2, 5:70],
              wide.half()[:, 1:78], wide[:0]):
        q, same = quantize(x), quantize(x.contiguous())
        assert torch.equal(q.codes, same.codes) and torch.equal(q.scales, same.scales)
        assert q.shape == x.shape and torch.equal(q.dequantize(), same.dequantize())


def test_parts_given_and_refusals():
    x = torch.randn(4, 70, device='cuda')
    q = quantize(x)
    # codes that begin at an odd byte, and scales: copied
    codes = torch.zeros(4 * 48 + 1, dtype=torch.uint8, device='cuda')[1:].view(4, 48)
    scales = torch.zeros(4 * 4 + 1, dtype=torch.uint8, device='cuda')[1:].view(4, 4)
    codes.copy_(q.codes), scales.copy_(q.scales)
    same = Microscaled(codes, scales, 70, torch.float32)
    assert torch.equal(same.dequantize(), q.dequantize())
    assert Microscaled(q.codes, q.scales, 70).dtype == torch.bfloat16
    for bad in (lambda: quantize(x.cpu()), lambda: quantize(x.double()), lambda: quantize(x[0]), lambda: quantize(x[:, :0]),
                lambda: quantize([1.0]), lambda: Microscaled(q.codes, q.scales, 100), lambda: Microscaled(q.codes, q.scales, 0),
                lambda: Microscaled(q.codes, q.scales[:, :3], 70), lambda: Microscaled(q.codes[:3], q.scales, 70),
                lambda: Microscaled(q.codes.cpu(), q.scales.cpu(), 70), lambda: Microscaled(q.codes.int(), q.scales, 70),
                lambda: Microscaled(q.codes, q.scales, 70, torch.int8), lambda: Microscaled(q.codes, q.scales, 70.0),
                lambda: q.dequantize(torch.float64)):
        with pytest.raises(ValueError):
            bad()
