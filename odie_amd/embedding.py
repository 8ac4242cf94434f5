"""Rows of a table by id on the GPU, scaled, with the table's gradient by sorted ids (odie_embed_forward /
odie_embed_backward): a code per tile, image or expert.  There is no CPU path."""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .rows import DTYPES, check_rows, pitch, records, row_major


def embed(table, ids, scale=1.0):
    """scale * table[ids] for table [rows, width] (CUDA fp32, fp16 or bf16) and integer ids of any shape
    (CUDA int32 or int64); zeros, and no gradient, for an id outside the table."""
    table = check_rows('table', table)
    if table.shape[0] == 0:
        raise ValueError('table must have at least one row')
    if (not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int32, torch.int64)
            or ids.device != table.device):
        raise ValueError('ids must be a CUDA int32 or int64 tensor on the table\'s device')
    ids = ids.contiguous()
    if records(table):
        return _Embed.apply(table, ids, float(scale))
    return _forward(table, ids, float(scale))


def _forward(table, ids, scale):
    out = torch.empty((*ids.shape, table.shape[1]), dtype=table.dtype, device=table.device)
    _lib.call('odie_embed_forward', table, table.data_ptr(), pitch(table), table.shape[0], ids.data_ptr(),
              ids.element_size(), ids.numel(), scale, table.shape[1], DTYPES[table.dtype], out.data_ptr())
    return out


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.shape, ctx.dtype = scale, table.shape, table.dtype
        return _forward(table, ids, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        ids, = ctx.saved_tensors
        vocab, width = ctx.shape
        rows = row_major(upstream.reshape(-1, width))
        dtype = DTYPES[ctx.dtype]
        dtable = torch.empty((vocab, width), dtype=ctx.dtype, device=ids.device)
        scratch = _lib.scratch('odie_embed_workspace', ids, ids.numel(), vocab, width, dtype)
        _lib.call('odie_embed_backward', ids, rows.data_ptr(), pitch(rows), ids.data_ptr(), ids.element_size(),
                  ids.numel(), vocab, ctx.scale, width, dtype, dtable.data_ptr(), _lib.ptr(scratch),
                  0 if scratch is None else scratch.numel())
        return dtable, None, None
