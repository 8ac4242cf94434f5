"""A learned router over experts or classes on the GPU: the choice of each row's experts with their softmax weights
(odie_choose_*), the loss that keeps the experts' load even (odie_balance_*), and the divergence from a teacher's
top logits (odie_distill_*), each with its gradient.  There is no CPU path.

  logits  = linear(x, router)                       [N, experts]
  expert, weights = choose(logits, choices)         for expert_order and combine of odie_amd.mixture
  loss, counts = balance(logits, expert)

A logit of -inf is masked: its expert is never chosen and has no share.  NaN and +inf make their row's softmax NaN.
"""
import numbers

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .rows import DTYPES, check_rows, pitch, records


def choose(logits, choices, *, normalize=True):
    """expert int32 [N, choices] and weights fp32 [N, choices] of logits [N, experts] (CUDA fp32, fp16 or bf16): each
    row's largest logits from the largest on, the lowest index first among equal ones, and their softmax over
    the row's chosen experts, or with normalize=False over all of them.  Where a row has fewer logits
    above -inf, the rest are -1 with weight 0.  At most 64 choices and 32768 experts."""
    logits = check_rows('logits', logits)
    if not isinstance(choices, numbers.Integral) or not 1 <= choices <= min(64, logits.shape[1]):
        raise ValueError('choices must be a whole number within 1..64 and the experts')
    if records(logits):
        return _Choose.apply(logits, int(choices), bool(normalize))
    return _choose(logits, int(choices), bool(normalize), None)


def balance(logits, expert):
    """The balance loss (fp32, no dimensions) of logits [N, experts] and the experts chosen for each row, expert int32
    [N, choices], and the entries of each expert, int32 [experts]:

      loss = experts * sum over e of (share of the entries that are e) * (mean over rows of softmax(logits)[e])

    It is 1 where both are even.  Entries outside 0..experts-1 are none, and rows of none (a batch's padding) take
    no part, whatever their logits are: the mean is over the others, and the loss of none at all is 0.  A row whose
    logits are all -inf has shares of 0."""
    logits = check_rows('logits', logits)
    if (not isinstance(expert, torch.Tensor) or expert.dtype != torch.int32 or expert.ndim != 2
            or expert.device != logits.device or expert.shape[0] != logits.shape[0] or expert.shape[1] == 0):
        raise ValueError('expert must be int32 [%d, choices] on the logits\' device' % logits.shape[0])
    expert = expert.contiguous()
    if records(logits):
        return _Balance.apply(logits, expert)
    return _balance(logits, expert, False)[:2]


def distill(logits, ids, teacher, *, temperature=1.0):
    """Each row's divergence from its teacher, fp32 [N]: sum over j of q_j (log q_j - log p[ids_j]) for logits
    [N, classes], where p = softmax(logits / temperature), ids (int32 or int64, [N, top]) are the teacher's classes
    and q the softmax of teacher / temperature ([N, top], any floating dtype of the three) over them alone.

    An id outside 0..classes-1 or a teacher's -inf is no entry; a row without any has loss 0 and no gradient.
    The temperature is within 2^-100..2^100.  Entries of one class count each.  One entry a row is the cross entropy
    of that class.  A row whose logits are all -inf has p = 0 and, with an entry, an infinite loss.  The teacher is
    fixed: it takes no gradient."""
    logits = check_rows('logits', logits)
    n, device = logits.shape[0], logits.device
    if (not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int32, torch.int64) or ids.ndim != 2
            or ids.device != device or ids.shape[0] != n or not 1 <= ids.shape[1] <= 1024):
        raise ValueError('ids must be int32 or int64 [%d, top] on the logits\' device, top at most 1024' % n)
    if (not isinstance(teacher, torch.Tensor) or teacher.dtype not in DTYPES or teacher.shape != ids.shape
            or teacher.device != device):
        raise ValueError('teacher must be fp32, fp16 or bf16 of the shape and device of ids')
    if records(teacher):
        raise ValueError('teacher takes no gradient: detach it')
    if not isinstance(temperature, numbers.Real) or not 2.0 ** -100 <= temperature <= 2.0 ** 100:
        raise ValueError('temperature must be a number within 2^-100..2^100')
    ids, teacher = ids.contiguous(), teacher.contiguous()
    if records(logits):
        return _Distill.apply(logits, ids, teacher, float(temperature))
    return _distill(logits, ids, teacher, float(temperature), None)


def _floats(logits, *shape):
    return logits.new_empty(shape, dtype=torch.float32)


def _choose(logits, choices, normalize, stats):
    n, experts = logits.shape
    expert = logits.new_empty((n, choices), dtype=torch.int32)
    weights = _floats(logits, n, choices)
    _lib.call('odie_choose_forward', logits, logits.data_ptr(), pitch(logits), n, experts, choices, int(normalize),
              DTYPES[logits.dtype], expert.data_ptr(), weights.data_ptr(), _lib.ptr(stats))
    return expert, weights


def _balance(logits, expert, keep):
    """loss, counts, and one buffer of: the norm, padding up to four, with `keep` the rows' statistics, the workspace."""
    n, experts = logits.shape
    choices = expert.shape[1]
    loss, counts = _floats(logits), logits.new_empty(experts, dtype=torch.int32)
    need = _lib.library().odie_balance_workspace(n, choices, experts)
    stats = 4 * n if keep else 0
    kept = _floats(logits, 4 + stats + max(need, 0) // 4)
    at = kept.data_ptr()
    _lib.call('odie_balance_forward', logits, logits.data_ptr(), pitch(logits), expert.data_ptr(), n, choices, experts,
              DTYPES[logits.dtype], loss.data_ptr(), counts.data_ptr(), at + 16 if keep else None, at,
              at + 16 + 4 * stats, need)
    return loss, counts, kept


def _distill(logits, ids, teacher, temperature, stats):
    n, classes = logits.shape
    loss = _floats(logits, n)
    dtype = DTYPES[logits.dtype]
    scratch = _lib.scratch('odie_distill_workspace', logits, n, classes, dtype)
    _lib.call('odie_distill_forward', logits, logits.data_ptr(), pitch(logits), ids.data_ptr(), ids.element_size(),
              teacher.data_ptr(), DTYPES[teacher.dtype], n, classes, ids.shape[1], temperature, dtype, loss.data_ptr(),
              _lib.ptr(stats), _lib.ptr(scratch), 0 if scratch is None else scratch.numel())
    return loss


class _Choose(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, choices, normalize):
        stats = None if normalize else _floats(logits, logits.shape[0], 2)
        expert, weights = _choose(logits, choices, normalize, stats)
        ctx.mark_non_differentiable(expert)
        # normalised weights have their gradient without the logits
        ctx.save_for_backward(expert, weights, None if normalize else logits, stats)
        ctx.shape, ctx.dtype = logits.shape, logits.dtype
        return expert, weights

    @staticmethod
    @once_differentiable
    def backward(ctx, _, upstream):
        expert, weights, logits, stats = ctx.saved_tensors
        n, experts = ctx.shape
        upstream = upstream.contiguous()
        dlogits = torch.empty((n, experts), dtype=ctx.dtype, device=weights.device)
        _lib.call('odie_choose_backward', weights, upstream.data_ptr(), expert.data_ptr(), weights.data_ptr(),
                  _lib.ptr(logits), 0 if logits is None else pitch(logits), _lib.ptr(stats), n, experts, expert.shape[1],
                  DTYPES[ctx.dtype], dlogits.data_ptr())
        return dlogits, None, None


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, expert):
        loss, counts, kept = _balance(logits, expert, True)
        ctx.mark_non_differentiable(counts)
        ctx.save_for_backward(logits, counts, kept)
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream, _):
        logits, counts, kept = ctx.saved_tensors
        n, experts = logits.shape
        upstream = upstream.contiguous()
        dlogits = logits.new_empty((n, experts))
        _lib.call('odie_balance_backward', logits, upstream.data_ptr(), logits.data_ptr(), pitch(logits),
                  counts.data_ptr(), kept.data_ptr() + 16, kept.data_ptr(), n, experts, DTYPES[logits.dtype],
                  dlogits.data_ptr())
        return dlogits, None


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, temperature):
        stats = _floats(logits, logits.shape[0], 4)
        loss = _distill(logits, ids, teacher, temperature, stats)
        ctx.save_for_backward(logits, ids, teacher, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        logits, ids, teacher, stats = ctx.saved_tensors
        n, classes = logits.shape
        upstream = upstream.contiguous()
        dlogits = logits.new_empty((n, classes))
        _lib.call('odie_distill_backward', logits, upstream.data_ptr(), logits.data_ptr(), pitch(logits), ids.data_ptr(),
                  ids.element_size(), teacher.data_ptr(), DTYPES[teacher.dtype], stats.data_ptr(), n, classes,
                  ids.shape[1], ctx.temperature, DTYPES[logits.dtype], dlogits.data_ptr())
        return dlogits, None, None, None
