"""Shared rows: lookup with scaling, and the table's gradient summed by row (gsx_b200_embedding_*)."""
from __future__ import annotations

import torch

from ._capi import OUT_OF_RANGE, GsxError, lib
from ._tensors import (FLOAT_TYPES, INDEX_TYPES, below_2_31, empty, invalid, launch, on_device, row_stride, type_code,
                       word)


def embedding_lookup(table, index, out=None, scale: float = 1.0, bad=None, stream=None):
    """out[n] = scale * table[index[n]] for a [rows, dim] table and an index tensor of any shape; out is
    index.shape + (dim,), of the table's type unless given (float32, float16 or bfloat16 each).  Rows may be
    strided.  An index outside the table sets the one-word tensor `bad` to 1 (where given) and leaves its row."""
    if table.dim() != 2:
        raise invalid("table must be [rows, dim]")
    rows, dim = table.shape
    device = table.device
    on_device(device, index, out, bad)
    if not index.is_contiguous():
        raise invalid("index must be contiguous")
    count = index.numel()
    if (rows | dim | count) >> 31:
        below_2_31(rows, dim, count)
    if out is None:
        out = empty((*index.shape, dim), table.dtype, device, stream)
    elif out.shape[:-1] != index.shape or out.shape[-1:] != table.shape[1:]:
        raise invalid(f"out must be {(*index.shape, dim)}, not {tuple(out.shape)}")
    launch(lib().gsx_b200_embedding_lookup, device, stream, table.data_ptr(), type_code(table, FLOAT_TYPES, "table"),
           rows, dim, dim if table.is_contiguous() else row_stride(table, dim, "table"), index.data_ptr(),
           type_code(index, INDEX_TYPES, "index"), count, scale, out.data_ptr(), type_code(out, FLOAT_TYPES, "out"),
           dim if out.is_contiguous() else row_stride(out, dim, "out"), None if bad is None else word(bad, "bad"))
    return out


def embedding_backward(grad_out, index, grad_table, scale: float = 1.0, padding_row: int | None = None,
                       accumulate: bool = False, bad=None, stream=None):
    """grad_table[v] = scale * sum of grad_out[n] over index[n] = v, written for every row (added to it when
    accumulate), in f32 sums.  Their order depends on the sizes, types, alignment and strides only: the same call
    gives the same bits.  grad_out is index.shape + (dim,), grad_table [rows, dim].  Indices equal to padding_row take no part; out-of-range ones set `bad`."""
    if grad_table.dim() != 2:
        raise invalid("grad_table must be [rows, dim]")
    rows, dim = grad_table.shape
    device = grad_table.device
    on_device(device, grad_out, index, bad)
    if not index.is_contiguous():
        raise invalid("index must be contiguous")
    count = index.numel()
    if (rows | dim | count) >> 31:
        below_2_31(rows, dim, count)
    if grad_out.shape[:-1] != index.shape or grad_out.shape[-1:] != grad_table.shape[1:]:
        raise invalid(f"grad_out must be {(*index.shape, dim)}, not {tuple(grad_out.shape)}")
    if padding_row is None:
        padding_row = -1
    elif not 0 <= padding_row < rows:
        raise GsxError(OUT_OF_RANGE, "padding_row must be a row of grad_table")
    L = lib()
    size = L.gsx_b200_embedding_workspace_bytes(count, rows, dim)
    workspace = empty((size,), torch.uint8, device, stream)
    launch(L.gsx_b200_embedding_backward, device, stream, grad_out.data_ptr(),
           type_code(grad_out, FLOAT_TYPES, "grad_out"), row_stride(grad_out, dim, "grad_out"), index.data_ptr(),
           type_code(index, INDEX_TYPES, "index"), count, scale, padding_row, grad_table.data_ptr(),
           type_code(grad_table, FLOAT_TYPES, "grad_table"), rows, dim, row_stride(grad_table, dim, "grad_table"),
           1 if accumulate else 0, workspace.data_ptr(), size, word(bad, "bad"))
    return grad_table
