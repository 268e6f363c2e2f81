"""Keeping the Gaussians of a scene, or the rows of key-value caches, within a budget by accumulated weight
(gsx_b200_budget_*).

A score tensor is [length] for one set of entries (a scene) or [.., length] for several (one per batch entry and
head); `lengths`, where given, is an int32 tensor of the leading shape with the entries in use."""
from __future__ import annotations

import ctypes

import torch

from ._capi import GATHER_MAX_FIELDS, NOT_SUPPORTED, OUT_OF_RANGE, GsxError, lib
from ._tensors import FLOAT_TYPES, below_2_31, empty, group_stride, invalid, launch, on_device, type_code, word


def _score(score, name="score"):
    """(groups, length, stride between groups) of a score tensor."""
    if score.dim() < 1 or score.dtype != torch.float32:
        raise invalid(f"{name} must be a float32 tensor of at least one dimension")
    length = score.shape[-1]
    groups = score.shape[:-1].numel()
    if score.is_contiguous():
        return groups, length, length
    if length > 1 and score.stride(-1) != 1:
        raise invalid(f"the last dimension of {name} must be contiguous")
    return groups, length, group_stride(score, score.dim() - 1, name) if groups > 1 else length


def _per_group(t, lead, name):
    """Pointer of an int32 tensor with one value per group (None allowed)."""
    if t is None:
        return None
    if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() != lead.numel():
        raise invalid(f"{name} must be a contiguous int32 tensor with one value per group")
    return t.data_ptr()


def budget_accumulate(score, weights, out=None, decay: float = 1.0, lengths=None, row_lengths=None, stream=None):
    """out[.., j] = decay * score[.., j] + sum over r of weights[.., r, j] for the entries in use; the others are
    copied.  weights is score's leading shape + (rows, length), float32, float16 or bfloat16; row_lengths (int32,
    one per group) leaves the rows behind it out.  out None: score is updated in place.  decay 0 starts anew."""
    groups, length, stride = _score(score)
    lead = score.shape[:-1]
    if out is None:
        out = score
    elif out.shape != score.shape:
        raise invalid("out must have score's shape")
    device = score.device
    on_device(device, weights, out, lengths, row_lengths)
    if weights.dim() != score.dim() + 1 or weights.shape[:-2] != lead or weights.shape[-1] != length:
        raise invalid(f"weights must be {(*lead, 'rows', length)}, not {tuple(weights.shape)}")
    rows = weights.shape[-2]
    if length > 1 and weights.stride(-1) != 1:
        raise invalid("the last dimension of weights must be contiguous")
    if (groups | rows | length) >> 31:
        below_2_31(groups, rows, length)
    if weights.is_contiguous():
        group_step, row_step = rows * length, length
    else:
        group_step = group_stride(weights, weights.dim() - 2, "weights")
        row_step = weights.stride(-2) if rows > 1 else length
    launch(lib().gsx_b200_budget_accumulate, device, stream, score.data_ptr(), stride, weights.data_ptr(),
           type_code(weights, FLOAT_TYPES, "weights"), group_step, row_step, groups, rows, length,
           None if lengths is None else _per_group(lengths, lead, "lengths"),
           None if row_lengths is None else _per_group(row_lengths, lead, "row_lengths"), decay, out.data_ptr(),
           length if out.is_contiguous() and out.dtype == torch.float32 else _score(out, "out")[2])
    return out


def budget_select(score, budget: int, lengths=None, first: int = 0, recent: int = 0, keep=None, kept=None, drop=None,
                  stream=None):
    """(keep, kept): per group the increasing list of the entries that stay within `budget` (the `first` first,
    the `recent` last, and the largest scores of the others, ties to the lowest index; NaN is below every number)
    and its length min(entries in use, budget).  keep is int32, leading shape + (at least min(budget, length),);
    drop, where given, int32 of score's shape, receives the others.  Places behind the lists are left as they were.
    No output may overlap another or an input (kept is not lengths updated in place)."""
    groups, length, stride = _score(score)
    lead = score.shape[:-1]
    if (groups | length | budget) >> 31:
        below_2_31(groups, length, budget)
    if first < 0 or recent < 0:
        raise GsxError(OUT_OF_RANGE, "first and recent must not be negative")
    if first + recent > budget:
        raise invalid("first + recent must be at most budget")
    device = score.device
    on_device(device, lengths, keep, kept, drop)
    most = min(budget, length)
    if keep is None:
        keep = empty((*lead, most), torch.int32, device, stream)
    elif keep.dtype != torch.int32 or not keep.is_contiguous() or keep.shape[:-1] != lead or keep.shape[-1] < most:
        raise invalid(f"keep must be a contiguous int32 tensor of shape {(*lead, most)} or wider")
    if kept is None:
        kept = empty(lead, torch.int32, device, stream)
    if drop is not None and (drop.dtype != torch.int32 or not drop.is_contiguous() or drop.shape != score.shape):
        raise invalid("drop must be a contiguous int32 tensor of score's shape")
    L = lib()
    size = L.gsx_b200_budget_workspace_bytes(groups, length)
    workspace = empty((size,), torch.uint8, device, stream) if size else None
    launch(L.gsx_b200_budget_select, device, stream, score.data_ptr(), stride, groups, length,
           None if lengths is None else _per_group(lengths, lead, "lengths"), first, recent, budget, keep.data_ptr(),
           keep.shape[-1],
           _per_group(kept, lead, "kept"), None if drop is None else drop.data_ptr(), length,
           None if workspace is None else workspace.data_ptr(), size)
    return keep, kept


def _field(t, lead, tail, side):
    """Entries and (outer, inner, row) strides in bytes of one side of a gather field; checks its shape."""
    n = len(lead)
    shape, size = t.shape, t.element_size()
    if len(shape) <= n or shape[:n] != lead or shape[n + 1:] != tail:
        raise invalid(f"{side} must be {(*lead, 'entries', *tail)}, not {tuple(shape)}")
    entries = shape[n]
    if t.is_contiguous():
        row = tail.numel() * size
        inner = row * entries if n else 0
        return entries, inner * lead[1] if n == 2 else 0, inner, row
    want = 1
    for d in range(len(shape) - 1, n, -1):
        if shape[d] > 1 and t.stride(d) != want:
            raise invalid(f"the rows of {side} must be contiguous")
        want *= shape[d]
    return (entries, t.stride(0) * size if n == 2 else 0, t.stride(n - 1) * size if n else 0, t.stride(n) * size)


def budget_gather(fields, keep, kept, bad=None, stream=None):
    """Row r of dst = row keep[.., r] of src for r < kept[..], for every (src, dst) pair of `fields` (up to 32) in
    one launch.  keep is [budget], [heads, budget] or [batch, heads, budget]; src is its leading shape + (length,) +
    any row shape, dst the same with at least `budget` rows; both may be strided in all but the row, so a cache may
    be a transposed view.  Rows of dst behind kept are left as they were.  No dst may overlap a src, keep, kept or bad,
    and no row of a dst another one; several may interleave in one buffer."""
    lead = keep.shape[:-1]
    if keep.dim() < 1 or len(lead) > 2 or keep.dtype != torch.int32 or not keep.is_contiguous():
        raise invalid("keep must be a contiguous int32 tensor of one to three dimensions")
    if len(fields) > GATHER_MAX_FIELDS:
        raise GsxError(OUT_OF_RANGE, f"at most {GATHER_MAX_FIELDS} fields")
    device = keep.device
    on_device(device, kept, bad)
    budget = keep.shape[-1]
    n = len(lead)
    table, length = [], None
    for src, dst in fields:
        if src.device != device or dst.device != device:
            raise invalid(f"all tensors must be on {device}")
        if src.dtype != dst.dtype:
            raise GsxError(NOT_SUPPORTED, "src and dst must have the same type")
        tail = src.shape[n + 1:]
        entries, src_outer, src_inner, src_row = _field(src, lead, tail, "src")
        room, dst_outer, dst_inner, dst_row = _field(dst, lead, tail, "dst")
        if length is None:
            length = entries
        if entries != length or room < budget:
            raise invalid("every src must have the same number of entries, every dst at least keep's")
        # the members of gsx_b200_gather_field, all 64 bits wide
        table += (src.data_ptr(), dst.data_ptr(), tail.numel() * src.element_size(), src_outer, src_inner, src_row,
                  dst_outer, dst_inner, dst_row)
    outer, inner = ([1] * (2 - len(lead)) + list(lead))
    launch(lib().gsx_b200_budget_gather, device, stream, (ctypes.c_uint64 * len(table))(*table), len(fields), outer, inner, length or 0, budget,
           keep.data_ptr(), budget, _per_group(kept, lead, "kept"), word(bad, "bad"))
