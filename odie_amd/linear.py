"""Linear layers on the GPU: y = act(x W^T + b) + r in one launch, dense or with one matrix per expert over
rows sorted by expert, with every gradient through autograd (odie_linear_forward /
odie_linear_backward).  There is no CPU path.

Unlike the decoder and gate heads, whose shapes are fixed, a layer here has any width, an optional bias and
residual, one of six activations, and fp32, fp16 or bf16 tensors; sums are fp32, and the output is rounded once.
Between them, 16-bit layers round twice for the gradients: the sums before the activation, kept for its slope, and
the slope's product with the upstream, an operand of both matrix products.  Gradients of x and the weight
are then about 1.4 times as far from exact ones as a single rounding leaves them; fp32 layers round neither.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .rows import DTYPES, check_rows, pitch, records, row_major

ACTIVATIONS = ('none', 'relu', 'sigmoid', 'softplus', 'gelu', 'silu')   # their ODIE_ACT_ codes in order
_CODES = {name: code for code, name in enumerate(ACTIVATIONS)}


def linear(x, weight, bias=None, *, activation='none', residual=None, offsets=None):
    """act(x W^T + bias) + residual for x [N, inputs] (CUDA fp32, fp16 or bf16, as every other tensor).

    weight [outputs, inputs], bias [outputs]; or, with offsets (CUDA int32 [experts + 1],
    nondecreasing from 0, as ExpertGrid's or expert_order's), weight [experts, outputs, inputs] and
    bias [experts, outputs]: rows offsets[e]..offsets[e+1]-1 use expert e's, rows from offsets[experts]
    on have no expert, and get the residual alone or 0, and no gradient of their own.
    residual [N, outputs].  gelu is the exact one (by erf)."""
    if activation not in _CODES:
        raise ValueError('activation must be one of %s' % ', '.join(ACTIVATIONS))
    x = check_rows('x', x)
    n, inputs = x.shape
    lead = 1 if offsets is None else 2      # dimensions before the inputs
    if (not isinstance(weight, torch.Tensor) or weight.ndim != lead + 1 or weight.shape[-1] != inputs
            or weight.dtype != x.dtype or weight.device != x.device or weight.shape[0] == 0 or weight.shape[-2] == 0):
        raise ValueError('weight must be %s of x\'s dtype and device' %
                         ('[outputs, inputs]' if offsets is None else '[experts, outputs, inputs]'))
    outputs, experts = weight.shape[-2], 1 if offsets is None else weight.shape[0]
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.shape != weight.shape[:-1]
                             or bias.dtype != x.dtype or bias.device != x.device):
        raise ValueError('bias must be %s of x\'s dtype and device' %
                         ('[outputs]' if offsets is None else '[experts, outputs]'))
    if residual is not None:
        residual = check_rows('residual', residual, outputs, dtype=x.dtype, device=x.device, count=n)
    if offsets is not None:
        if (not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int32 or offsets.ndim != 1
                or offsets.numel() != experts + 1 or offsets.device != x.device):
            raise ValueError('offsets must be a CUDA int32 tensor of experts + 1 entries')
        offsets = offsets.contiguous()
    if records(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, offsets, _CODES[activation])
    return _forward(x, weight.contiguous(), None if bias is None else bias.contiguous(), residual, offsets,
                    _CODES[activation], None)


def _forward(x, weight, bias, residual, offsets, activation, pre):
    n, outputs = x.shape[0], weight.shape[-2]
    out = torch.empty((n, outputs), dtype=x.dtype, device=x.device)
    _lib.call('odie_linear_forward', x, x.data_ptr(), pitch(x), n, weight.data_ptr(), _lib.ptr(bias),
              _lib.ptr(residual), 0 if residual is None else pitch(residual), _lib.ptr(offsets),
              1 if offsets is None else weight.shape[0], x.shape[1], outputs, DTYPES[x.dtype], activation,
              out.data_ptr(), outputs, _lib.ptr(pre))
    return out


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, offsets, activation):
        weight = weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        want_x, want_weight, want_bias = ctx.needs_input_grad[:3]
        computed = want_x or want_weight or want_bias       # the residual's gradient is the upstream itself
        # the sums before the activation, from which the backward takes its slope
        keep = activation and computed
        pre = torch.empty((x.shape[0], weight.shape[-2]), dtype=x.dtype, device=x.device) if keep else None
        out = _forward(x, weight, bias, residual, offsets, activation, pre)
        # what the wanted gradients read
        ctx.save_for_backward(x if want_weight else None, weight if want_x else None, pre,
                              offsets if computed else None)
        ctx.activation, ctx.inputs, ctx.weights = activation, x.shape[1], weight.shape
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        x, weight, pre, offsets = ctx.saved_tensors
        want_x, want_weight, want_bias, want_residual = ctx.needs_input_grad[:4]
        dx = dweight = dbias = None
        if want_x or want_weight or want_bias:
            rows = row_major(upstream)
            n, inputs = rows.shape[0], ctx.inputs
            outputs, experts = rows.shape[1], 1 if offsets is None else ctx.weights[0]
            dtype = DTYPES[rows.dtype]
            dx = rows.new_empty((n, inputs)) if want_x else None
            dweight = rows.new_empty(ctx.weights) if want_weight else None
            dbias = rows.new_empty(ctx.weights[:-1]) if want_bias else None
            scratch = _lib.scratch('odie_linear_workspace', rows, n, experts, int(offsets is not None), inputs, outputs,
                                   dtype, ctx.activation, int(want_weight), int(want_bias))
            _lib.call('odie_linear_backward', rows, rows.data_ptr(), pitch(rows), _lib.ptr(x),
                      0 if x is None else pitch(x), _lib.ptr(pre), n, _lib.ptr(weight), _lib.ptr(offsets), experts, inputs, outputs, dtype,
                      ctx.activation, _lib.ptr(dx), _lib.ptr(dweight), _lib.ptr(dbias), _lib.ptr(scratch),
                      0 if scratch is None else scratch.numel())
        return dx, dweight, dbias, upstream if want_residual else None, None, None
