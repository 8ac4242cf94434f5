"""Microscaled 4-bit floating point on the GPU: tensors quantised in blocks of 32 values along the last dimension
(odie_mx_quantize / odie_mx_dequantize), for the weights of odie_amd.linear.linear and the rows it multiplies.
There is no CPU path.

A value is +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times its block's scale, a power of two: 4.25 bits a value.  The
largest magnitude of a block is scaled into [4, 8) and clamped at 6; values are rounded to nearest even: off by at most a
quarter of themselves from 1/4 of the largest on, which is one scale at least, and below one scale by a quarter of the
scale.
"""
import math

import torch

from . import _lib
from .rows import DTYPES, pitch, row_major, tangents

BLOCK = 32


def _blocks(width):
    return (width + BLOCK - 1) // BLOCK


class Microscaled:
    """A tensor [..., width] in 4 bits.  codes uint8 [..., 16 * blocks], blocks = ceil(width / 32): two values a byte, the
    first in the low half, each sign, two bits of exponent and one of fraction, 0 past the width; scales uint8 [...,
    blocks rounded up to a multiple of 4]: 2^(scale - 127), 255 for NaN, 0 past the last block.  dtype (fp32, fp16 or
    bf16): of the tensor it stands for, and of what is computed from it.  Both are taken as they are, or
    copied where they are not contiguous and aligned.  shape, ndim and device are the tensor's."""

    def __init__(self, codes, scales, width, dtype=torch.bfloat16):
        if (not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor) or codes.dtype != torch.uint8
                or scales.dtype != torch.uint8 or not codes.is_cuda or codes.device != scales.device
                or codes.ndim not in (2, 3) or codes.shape[:-1] != scales.shape[:-1]):
            raise ValueError('codes and scales must be CUDA uint8 tensors of two or three dimensions on one device')
        if (isinstance(width, bool) or not isinstance(width, int) or not 1 <= width <= 1 << 20
                or codes.shape[-1] != 16 * _blocks(width) or scales.shape[-1] != (_blocks(width) + 3) // 4 * 4):
            raise ValueError('codes must have 16 bytes and scales one for each block of 32 of the width, the scales in '
                             'whole fours')
        if dtype not in DTYPES:
            raise ValueError('dtype must be fp32, fp16 or bf16')
        self._hold(_aligned(codes, 16), _aligned(scales, 4), width, dtype, (*codes.shape[:-1], width))

    def _hold(self, codes, scales, width, dtype, shape):
        self.codes, self.scales, self.width, self.dtype = codes, scales, width, dtype
        self.shape, self.ndim, self.device = torch.Size(shape), len(shape), codes.device

    def dequantize(self, dtype=None):
        """The tensor of dtype (its own if not given), rounded where that does not hold a value."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in DTYPES:
            raise ValueError('dtype must be fp32, fp16 or bf16')
        out = self.codes.new_empty(self.shape, dtype=dtype)
        _lib.call('odie_mx_dequantize', self.codes, self.codes.data_ptr(), self.scales.data_ptr(),
                  math.prod(self.shape[:-1]), self.width, DTYPES[dtype], out.data_ptr(), self.width)
        return out


def _aligned(value, bytes):
    value = value.contiguous()
    return value if value.data_ptr() % bytes == 0 else value.clone()


def quantize(x):
    """x (CUDA fp32, fp16 or bf16, [N, width] or [experts, outputs, width]) as Microscaled.  A block that holds a NaN or
    an infinity becomes NaN.  The result is whole numbers: no gradient passes through them, and x may not carry a tangent."""
    if not isinstance(x, torch.Tensor) or x.dtype not in DTYPES or x.ndim not in (2, 3) or not x.is_cuda:
        raise ValueError('x must be a CUDA fp32, fp16 or bf16 tensor of two or three dimensions')
    *lead, width = x.shape
    if not 1 <= width <= 1 << 20:
        raise ValueError('x must have 1 to 2^20 columns')
    if tangents(x):
        raise NotImplementedError('quantize has no forward-mode derivative')
    rows = row_major(x if x.ndim == 2 else x.detach().reshape(-1, width))
    blocks = _blocks(width)
    codes = x.new_empty((*lead, 16 * blocks), dtype=torch.uint8)
    scales = x.new_empty((*lead, (blocks + 3) // 4 * 4), dtype=torch.uint8)
    _lib.call('odie_mx_quantize', rows, rows.data_ptr(), pitch(rows), rows.shape[0], width, DTYPES[x.dtype],
              codes.data_ptr(), scales.data_ptr())
    made = Microscaled.__new__(Microscaled)     # nothing to check
    made._hold(codes, scales, width, x.dtype, (*lead, width))
    return made
