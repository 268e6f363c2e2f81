"""Host-side refusals of the embedding and budget entry points, through the C ABI (no GPU: nothing is launched)."""
import ctypes

import pytest
import torch

import gsx_b200 as gb
from gsx_b200 import _capi

P = 4096  # an aligned non-null address: every call here returns before it is used
F32, F16, BF16, U8, I32, I64 = 0, 1, 2, 8, 12, 13


def _lookup(table=1 << 20, ttype=F32, rows=4, dim=8, tstride=8, index=1 << 16, itype=I32, count=3, out=P, otype=F32, ostride=8):
    return _capi.lib().gsx_b200_embedding_lookup(table, ttype, rows, dim, tstride, index, itype, count, 1.0, out, otype,
                                                 ostride, None, None)


def _backward(grad=1 << 20, gtype=F32, gstride=8, index=1 << 16, itype=I32, count=3, padding=-1, scale=1.0, table=P, ttype=F32, rows=4, dim=8,
              tstride=8, ws=P, size=1 << 40):
    return _capi.lib().gsx_b200_embedding_backward(grad, gtype, gstride, index, itype, count, scale, padding, table, ttype,
                                                   rows, dim, tstride, 0, ws, size, None, None)


def _accumulate(score=P, sstride=16, w=1 << 20, wtype=F32, gstride=32, rstride=16, groups=2, rows=2, length=16, out=P,
                ostride=16):
    return _capi.lib().gsx_b200_budget_accumulate(score, sstride, w, wtype, gstride, rstride, groups, rows, length, None,
                                                  None, 1.0, out, ostride, None)


def _select(score=P, sstride=16, groups=2, length=16, first=0, recent=0, budget=8, keep=P, kstride=8, kept=P, drop=None,
            dstride=0, ws=None, size=0):
    return _capi.lib().gsx_b200_budget_select(score, sstride, groups, length, None, first, recent, budget, keep, kstride,
                                              kept, drop, dstride, ws, size, None)


def _gather(fields=None, count=1, outer=1, inner=1, length=16, budget=8, keep=P, kstride=8, kept=P, **field):
    if fields is None:
        f = dict(src=P, dst=1 << 20, row_bytes=12, src_row_stride=12, dst_row_stride=12, **{})
        f.update(field)
        fields = (_capi.GatherField * 1)(_capi.GatherField(**f))
    return _capi.lib().gsx_b200_budget_gather(fields, count, outer, inner, length, budget, keep, kstride, kept, None, None)


CASES = [
    (gb.NOT_SUPPORTED, _lookup, [dict(ttype=U8), dict(otype=I32), dict(itype=F32)]),
    (gb.OUT_OF_RANGE, _lookup, [dict(rows=2 ** 31), dict(count=2 ** 31), dict(tstride=2 ** 41), dict(tstride=2 ** 30),
                                dict(count=2 ** 30, dim=2 ** 30, tstride=2 ** 30, ostride=2 ** 30)]),
    (gb.INVALID_ARGUMENT, _lookup, [dict(table=None), dict(index=None), dict(out=None), dict(tstride=7), dict(ostride=7),
                                    dict(table=(1 << 20) + 2), dict(out=P + 1, otype=F16), dict(index=(1 << 16) + 4, itype=I64),
                                    dict(out=(1 << 20) + 64), dict(out=(1 << 20) - 32), dict(out=(1 << 16) - 64)]),
    (_capi.SUCCESS, _lookup, [dict(count=0), dict(dim=0)]),
    (gb.NOT_SUPPORTED, _backward, [dict(gtype=U8), dict(ttype=I32), dict(itype=U8)]),
    (gb.OUT_OF_RANGE, _backward, [dict(rows=2 ** 31), dict(padding=4), dict(gstride=2 ** 30),
                                  dict(dim=2 ** 22, gstride=2 ** 22, tstride=2 ** 22)]),
    (gb.INVALID_ARGUMENT, _backward, [dict(grad=None), dict(index=None), dict(table=None), dict(ws=None), dict(gstride=7),
                                      dict(tstride=7), dict(size=100), dict(ws=P + 8), dict(grad=(1 << 20) + 2),
                                      dict(scale=float('inf')), dict(scale=float('nan')), dict(table=(1 << 20) - 64),
                                      dict(table=(1 << 16) - 64),
                                      dict(rows=0)]),
    (_capi.SUCCESS, _backward, [dict(dim=0), dict(rows=0, count=0)]),
    (gb.NOT_SUPPORTED, _accumulate, [dict(wtype=U8)]),
    (gb.OUT_OF_RANGE, _accumulate, [dict(groups=2 ** 31), dict(rows=2 ** 31), dict(length=2 ** 31), dict(gstride=2 ** 41)]),
    (gb.INVALID_ARGUMENT, _accumulate, [dict(score=None), dict(out=None), dict(w=None), dict(sstride=15), dict(ostride=15),
                                        dict(rstride=15), dict(score=P + 2), dict(out=P + 4), dict(out=P + 64),
                                        dict(w=P + 64), dict(ostride=17)]),
    (_capi.SUCCESS, _accumulate, [dict(groups=0), dict(length=0)]),
    (gb.OUT_OF_RANGE, _select, [dict(groups=2 ** 31), dict(length=2 ** 31), dict(budget=2 ** 31),
                                dict(groups=70_000, length=400_000, sstride=400_000), dict(groups=2 ** 28)]),
    (gb.INVALID_ARGUMENT, _select, [dict(first=9), dict(first=4, recent=5), dict(recent=2 ** 64 - 1), dict(score=None),
                                    dict(keep=None), dict(kept=None), dict(sstride=15), dict(kstride=7),
                                    dict(drop=P, dstride=15), dict(score=P + 1), dict(keep=P + 2),
                                    dict(length=400_000, sstride=400_000),
                                    dict(length=400_000, sstride=400_000, ws=P, size=100),
                                    dict(length=400_000, sstride=400_000, ws=P + 1, size=1 << 30)]),
    (_capi.SUCCESS, _select, [dict(groups=0)]),
    (gb.OUT_OF_RANGE, _gather, [dict(count=33), dict(count=-1), dict(outer=2 ** 16, inner=2 ** 16), dict(length=2 ** 31),
                                dict(src_row_stride=2 ** 32), dict(src_outer_stride=2 ** 43), dict(row_bytes=2 ** 32, dst_row_stride=2 ** 32)]),
    (gb.INVALID_ARGUMENT, _gather, [dict(keep=None), dict(kept=None), dict(src=None), dict(dst=None),
                                    dict(dst_row_stride=11), dict(dst=P + 180), dict(dst=P - 12 * 7),
                                    dict(inner=2, kstride=7), dict(keep=P + 2), dict(kept=P + 1)]),
    (_capi.SUCCESS, _gather, [dict(count=0), dict(outer=0), dict(budget=0), dict(row_bytes=0)]),
]


@pytest.mark.parametrize("code,call,kw", [(c, f, k) for c, f, ks in CASES for k in ks])
def test_refused_before_any_launch(code, call, kw):
    assert call(**kw) == code
    if code:
        assert _capi.lib().gsx_b200_last_error()


def test_workspace_sizes():
    L = _capi.lib()
    assert L.gsx_b200_embedding_workspace_bytes(10, 0, 4) == 0
    small = L.gsx_b200_embedding_workspace_bytes(100, 50, 4)
    assert 800 <= small < 1 << 20
    # a table that fits shared memory: one table of sums for each of up to 296 chunks
    assert L.gsx_b200_embedding_workspace_bytes(500_000, 256, 8) == 256 + 296 * 256 * 8 * 4
    assert L.gsx_b200_embedding_workspace_bytes(500_000, 257, 8) == 256 + 296 * 257 * 8 * 4
    assert L.gsx_b200_embedding_workspace_bytes(3_000_000, 4096, 3) == 256 + 296 * 4096 * 3 * 4
    assert L.gsx_b200_embedding_workspace_bytes(1000, 10, 4) == 256 + 2 * 10 * 4 * 4
    # else (row, position) pairs: once for a sort of one pass (up to 256 rows), twice for more
    one = L.gsx_b200_embedding_workspace_bytes(500_000, 256, 1000)
    two = L.gsx_b200_embedding_workspace_bytes(500_000, 257, 1000)
    assert 4_000_000 <= two - one < 4_001_000
    assert L.gsx_b200_budget_workspace_bytes(32, 131_072) == 0
    assert 0 < L.gsx_b200_budget_workspace_bytes(32, 131_073) < 4 << 20


def test_python_calls_refuse_host_tensors():
    t, i = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int32)
    calls = [lambda: gb.embedding_lookup(t, i), lambda: gb.embedding_backward(torch.zeros(2, 3), i, t),
             lambda: gb.budget_accumulate(torch.zeros(3), torch.zeros(2, 3)), lambda: gb.budget_select(torch.zeros(3), 2),
             lambda: gb.budget_gather([(t, t)], i, i[0])]
    for call in calls:
        with pytest.raises(gb.GsxError) as e:
            call()
        assert e.value.code == gb.INVALID_ARGUMENT
