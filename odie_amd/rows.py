"""What the row operators (linear, mixture, embedding) share: their element types and the checks of
their tensors."""
import torch
from torch.autograd import forward_ad

from . import _lib

DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def check_rows(name, value, width=None, *, dtype=None, device=None, count=None):
    """value as rows the kernels read: CUDA fp32, fp16 or bf16 [count, width], each row contiguous (a
    tensor that is not is copied)."""
    if not isinstance(value, torch.Tensor) or value.dtype not in DTYPES or value.ndim != 2 or not value.is_cuda:
        raise ValueError('%s must be a CUDA fp32, fp16 or bf16 tensor of two dimensions' % name)
    if dtype is not None and value.dtype != dtype:
        raise ValueError('%s must have the dtype of the other tensors (%s)' % (name, dtype))
    if device is not None and value.device != device:
        raise ValueError('%s must be on the device of the other tensors (%s)' % (name, device))
    if (width is not None and value.shape[1] != width) or (count is not None and value.shape[0] != count):
        raise ValueError('%s must be [%s, %s]' % (name, 'N' if count is None else count,
                                                  'width' if width is None else width))
    if value.shape[1] == 0:
        raise ValueError('%s must have at least one column' % name)
    return row_major(value)


def row_major(value):
    """value, or its copy where a row is not contiguous or rows overlap."""
    n, width = value.shape
    if (width > 1 and value.stride(1) != 1) or (n > 1 and value.stride(0) < width):
        return value.contiguous()
    return value


def pitch(rows):
    """Elements from row to row of what row_major returned.  The stride of a single row means nothing and may be any
    number, also after contiguous()."""
    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


def tangents(*tensors):
    """Whether one of the tensors carries a tangent (forward mode, also without gradients)."""
    if forward_ad._current_level < 0:       # no level is open; asking each tensor costs more
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def records(*tensors):
    """Whether autograd has to see the call: it will ask for a gradient of one of the tensors, or one of them carries a
    tangent, which autograd refuses for these operators."""
    return tangents(*tensors) or torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
