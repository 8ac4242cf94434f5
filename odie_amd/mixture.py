"""Mixtures of experts on the GPU: rows sorted by expert, sent to their slots and brought back with weights,
and a decoder per expert between the two.  There is no CPU path.

Where the multi-expert step routes each pixel to the one expert of its tile, a row here goes to any
number of experts with a weight each: a blend over the borders of neighbouring tiles, or a learned router.

  order = expert_order(expert, experts)            expert [N, choices] -> slots and offsets (odie_sort)
  sent  = dispatch(x, order)                       [N * choices, width], sorted by expert
  ...   = linear(sent, W, b, offsets=order.offsets)
  y     = combine(rows, order, weights)            y[i] = sum_j weights[i, j] rows[slots[i, j]]

RoutedMixture has the learned router (odie_amd.router), and MicroscaledMixture keeps a mixture's layers in 4 bits
(odie_amd.microscale).
"""
import math
import numbers

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .embedding import embed
from .linear import ACTIVATIONS, linear
from .microscale import Microscaled, quantize
from .router import choose
from .rows import DTYPES, check_rows, pitch, records, row_major


class ExpertOrder:
    """Entries (row, choice) in a stable order by expert.  slots int32 [N, choices]: the sorted place of
    each entry, -1 where its expert is none; source int32 [N * choices]: the entry (row * choices +
    choice) of each sorted place; offsets int32 [experts + 1]: the places of each expert's entries, those
    without an expert follow from offsets[experts] on."""

    def __init__(self, slots, source, offsets, experts):
        self.slots, self.source, self.offsets, self.experts = slots, source, offsets, experts


def expert_order(expert, experts):
    """The order of expert (CUDA int32 or int64, [N] or [N, choices]): each entry's expert in
    [0, experts); any other value is no expert."""
    if (not isinstance(expert, torch.Tensor) or expert.dtype not in (torch.int32, torch.int64)
            or expert.ndim not in (1, 2) or not expert.is_cuda):
        raise ValueError('expert must be a CUDA int32 or int64 tensor, [N] or [N, choices]')
    if expert.ndim == 2 and expert.shape[1] == 0:
        raise ValueError('expert must have at least one choice a row')
    if not isinstance(experts, numbers.Integral) or experts < 1:
        raise ValueError('experts must be a whole number, at least 1')
    experts = int(experts)
    expert = expert.contiguous()
    n, device = expert.numel(), expert.device
    scratch = _lib.scratch('odie_sort_workspace', expert, n, experts)
    source = torch.empty(n, dtype=torch.int32, device=device)
    slots = torch.empty(expert.shape if expert.ndim == 2 else (n, 1), dtype=torch.int32, device=device)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=device)
    _lib.call('odie_sort', expert, expert.data_ptr(), expert.element_size(), n, experts, source.data_ptr(), None,
              slots.data_ptr(), offsets.data_ptr(), _lib.ptr(scratch), 0 if scratch is None else scratch.numel())
    return ExpertOrder(slots, source, offsets, experts)


def dispatch(x, order):
    """Rows x [N, width] at their slots: [N * choices, width] sorted by expert, zeros from
    offsets[experts] on."""
    x = check_rows('x', x, count=order.slots.shape[0], device=order.slots.device)
    return _Dispatch.apply(x, order) if records(x) else _dispatch(x, order)


def combine(rows, order, weights=None):
    """y[i] = sum over j of weights[i, j] * rows[slots[i, j]] for rows [N * choices, width] sorted by
    expert; weights [N, choices], 1 if not given.  Entries without an expert add nothing."""
    n, choices = order.slots.shape
    rows = check_rows('rows', rows, count=n * choices, device=order.slots.device)
    if weights is not None:
        if (not isinstance(weights, torch.Tensor) or weights.shape != order.slots.shape
                or not weights.is_floating_point() or weights.device != rows.device):
            raise ValueError('weights must be a floating-point tensor of the shape and device of order.slots')
        weights = weights.float().contiguous()
    return _Combine.apply(rows, weights, order) if records(rows, weights) else _combine(rows, order.slots, weights)


def _dispatch(x, order):
    n, choices = order.slots.shape
    out = torch.empty((n * choices, x.shape[1]), dtype=x.dtype, device=x.device)
    _lib.call('odie_rows_dispatch', x, x.data_ptr(), pitch(x), order.slots.data_ptr(), order.offsets.data_ptr(),
              n, choices, order.experts, x.shape[1], DTYPES[x.dtype], out.data_ptr())
    return out


def _combine(rows, slots, weights):
    n, choices = slots.shape
    out = torch.empty((n, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    _lib.call('odie_rows_combine', rows, rows.data_ptr(), pitch(rows), slots.data_ptr(), _lib.ptr(weights),
              n, choices, rows.shape[1], DTYPES[rows.dtype], out.data_ptr())
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.save_for_backward(order.slots)
        return _dispatch(x, order)

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        return _combine(row_major(upstream), ctx.saved_tensors[0], None), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order):
        want_rows, want_weights = ctx.needs_input_grad[:2]
        ctx.experts = order.experts
        # what the wanted gradients read
        ctx.save_for_backward(rows if want_weights else None, weights if want_rows else None, order.slots,
                              order.offsets if want_rows else None)
        return _combine(rows, order.slots, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        rows, weights, slots, offsets = ctx.saved_tensors
        want_rows, want_weights = ctx.needs_input_grad[:2]
        upstream = row_major(upstream)
        n, choices = slots.shape
        width = upstream.shape[1]
        drows = dweights = None
        if want_rows:
            drows = torch.empty((n * choices, width), dtype=upstream.dtype, device=upstream.device)
        if want_weights:
            dweights = torch.empty((n, choices), dtype=torch.float32, device=upstream.device)
        _lib.call('odie_rows_combine_backward', upstream, upstream.data_ptr(), pitch(upstream), _lib.ptr(rows),
                  0 if rows is None else pitch(rows), slots.data_ptr(), _lib.ptr(weights),
                  _lib.ptr(offsets), n, choices, ctx.experts, width, DTYPES[upstream.dtype], _lib.ptr(drows),
                  _lib.ptr(dweights))
        return drows, dweights, None


class ExpertMixture(nn.Module):
    """A two-layer decoder per expert, blended: y[i] = sum_j weights[i, j] D_e(x[i]), e = expert[i, j],
    D_e(x) = W2_e act(W1_e [x, code] + b1_e) + b2_e, where with `codes` > 0 a row's input is joined by the
    scaled code of its id (a table of `vocab` codes)."""

    def __init__(self, experts, inputs, hidden, outputs, *, activation='relu', codes=0, vocab=0, dtype=torch.float16,
                 device='cuda', seed=0):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError('activation must be one of %s' % ', '.join(ACTIVATIONS))
        if dtype not in DTYPES:
            raise ValueError('dtype must be fp32, fp16 or bf16')
        if (codes > 0) != (vocab > 0):
            raise ValueError('codes and vocab go together')
        self.experts, self.activation = int(experts), activation
        self.scale = math.sqrt(codes) if codes else 1.0
        generator = torch.Generator().manual_seed(seed)

        def uniform(*shape, bound):
            value = (2 * torch.rand(*shape, generator=generator) - 1) * bound
            return nn.Parameter(value.to(device=device, dtype=dtype))

        width = inputs + codes
        self.table = uniform(vocab, codes, bound=1.0 / codes) if codes else None
        self.weight1 = uniform(experts, hidden, width, bound=math.sqrt(6.0 / (width + hidden)))
        self.bias1 = uniform(experts, hidden, bound=0.0)
        self.weight2 = uniform(experts, outputs, hidden, bound=math.sqrt(6.0 / (hidden + outputs)))
        self.bias2 = uniform(experts, outputs, bound=0.0)

    def forward(self, x, expert, weights=None, ids=None):
        """x [N, inputs], expert [N, choices] (other values than 0..experts-1: none), weights [N, choices];
        ids [N] with codes.  Returns [N, outputs]."""
        return _blend(self, self.weight1, self.weight2, x, expert, weights, ids)

    def microscaled(self, *, rows=False):
        """A MicroscaledMixture of the parameters as they are now."""
        return MicroscaledMixture(self, rows=rows)


def _blend(mixture, weight1, weight2, x, expert, weights, ids, rows4=False):
    if (ids is None) != (mixture.table is None):
        raise ValueError('give ids exactly where the mixture has codes')
    if ids is not None:
        x = torch.cat((x, embed(mixture.table, ids, mixture.scale)), dim=1)
    order = expert_order(expert, mixture.experts)
    bits = quantize if rows4 else (lambda value: value)
    hidden = linear(bits(dispatch(x, order)), weight1, mixture.bias1, activation=mixture.activation, offsets=order.offsets)
    rows = linear(bits(hidden), weight2, mixture.bias2, offsets=order.offsets)
    return combine(rows, order, weights)


class MicroscaledMixture(nn.Module):
    """An ExpertMixture whose layers' weights are kept in 4 bits, 4.25 each with their scales: for serving it, or for
    training what lies before it (x and the router's weights get their gradients; the mixture's own parameters,
    copied here, are buffers).  With rows=True the rows that enter a layer are quantised to 4 bits too, and there is no
    gradient of x."""

    def __init__(self, mixture, *, rows=False):
        super().__init__()
        self.experts, self.activation, self.scale, self.rows = mixture.experts, mixture.activation, mixture.scale, bool(rows)
        self.dtype, self.widths = mixture.weight1.dtype, (mixture.weight1.shape[2], mixture.weight2.shape[2])
        for name in ('table', 'bias1', 'bias2'):
            value = getattr(mixture, name)
            self.register_buffer(name, None if value is None else value.detach().clone())
        for layer in (1, 2):
            weight = quantize(getattr(mixture, 'weight%d' % layer))
            self.register_buffer('codes%d' % layer, weight.codes)
            self.register_buffer('scales%d' % layer, weight.scales)

    def forward(self, x, expert, weights=None, ids=None):
        """As ExpertMixture.forward."""
        weight1, weight2 = (Microscaled(getattr(self, 'codes%d' % layer), getattr(self, 'scales%d' % layer),
                                        self.widths[layer - 1], self.dtype) for layer in (1, 2))
        if self.rows:
            if records(x):
                raise ValueError('rows of 4 bits have no backward: detach x')
        return _blend(self, weight1, weight2, x, expert, weights, ids, self.rows)


class RoutedMixture(nn.Module):
    """A mixture that chooses its experts itself: logits = x R^T, and each row's `choices` largest with their softmax
    weights (over the chosen, or with normalize=False over all) blend the experts' decoders.  The arguments are
    ExpertMixture's and choose's.  The logits are of x's type, fp32 sums rounded once; for a choice by fp32 ones beside
    16-bit layers: expert, weights = choose(linear(x.float(), m.router.float()), m.choices), m.mixture(x, expert, weights)."""

    def __init__(self, experts, choices, inputs, hidden, outputs, *, normalize=True, activation='relu', codes=0, vocab=0,
                 dtype=torch.float16, device='cuda', seed=0):
        super().__init__()
        self.mixture = ExpertMixture(experts, inputs, hidden, outputs, activation=activation, codes=codes, vocab=vocab,
                                     dtype=dtype, device=device, seed=seed)
        self.choices, self.normalize = int(choices), bool(normalize)
        generator = torch.Generator().manual_seed(seed + 1)
        value = torch.randn(experts, inputs, generator=generator) * inputs ** -0.5
        self.router = nn.Parameter(value.to(device=device, dtype=dtype))

    def forward(self, x, ids=None, allowed=None):
        """y [N, outputs], the router's logits [N, experts] (for balance and distill of odie_amd.router) and the chosen
        expert int32 [N, choices].  allowed (bool, [N, experts] or [experts]): where False, the expert is not
        chosen; a row without an allowed one gets zeros."""
        logits = linear(x, self.router)
        if allowed is not None:
            logits = logits.masked_fill(~allowed, -math.inf)
        expert, weights = choose(logits, self.choices, normalize=self.normalize)
        return self.mixture(x, expert, weights, ids), logits, expert
