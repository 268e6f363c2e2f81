"""Outputs that overlap one another or an input are refused before any launch (no GPU: nothing is launched), and the test
of strided sets of rows behind it agrees with a count of bytes."""
import ctypes
import os
import random
import subprocess

import pytest

import gsx_b200 as gb
from gsx_b200 import _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MB = 1 << 20  # pointers here are numbers: every call returns before one is used


@pytest.fixture(scope="module")
def spans(tmp_path_factory):
    at = tmp_path_factory.mktemp("spans")
    (at / "spans.cpp").write_text('''
#include "gsx_spans.h"
static GsxRows rows(const uint64_t *v)
{
    return GsxRows((const void *)(uintptr_t)v[0], v[1], { { v[2], v[3] }, { v[4], v[5] }, { v[6], v[7] } });
}
extern "C" int nested(const uint64_t *v) { return rows(v).nested(); }
extern "C" int meet(const uint64_t *a, const uint64_t *b) { return gsx_rows_meet(rows(a), rows(b)); }
''')
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{ROOT}/gsx_b200/csrc", str(at / "spans.cpp"), "-o",
                    str(at / "spans.so")], check=True)
    return ctypes.CDLL(str(at / "spans.so"))


def _c(v):
    return (ctypes.c_uint64 * 8)(*v)


def _bytes(v):
    at, size, c0, s0, c1, s1, c2, s2 = v
    places = [at + a * s0 + b * s1 + c * s2 + i for a in range(c0) for b in range(c1) for c in range(c2) for i in range(size)]
    return set(places), len(places)


def test_strided_rows_meet_where_their_bytes_do(spans):
    rng = random.Random(3)
    seen = {True: 0, False: 0}
    for _ in range(20_000):
        both = []
        for k in range(2):
            size, dims = rng.randint(1, 6), []
            extent = size
            for d in range(3):
                count, step = rng.randint(1, 4), extent + rng.randint(0, 12) if rng.random() < 0.8 else rng.randint(0, 30)
                if k and rng.random() < 0.5:
                    step = both[0][3 + 2 * d]
                dims.append((count, step))
                extent += (count - 1) * step
            rng.shuffle(dims)
            both.append([1000 + rng.randint(0, 60), size] + [x for d in dims for x in d])
        covered = [_bytes(v) for v in both]
        whole = [bool(spans.nested(_c(v))) for v in both]
        for (places, count), ok in zip(covered, whole):
            assert not ok or len(places) == count  # no byte in two places
        if all(whole):
            want = bool(covered[0][0] & covered[1][0])
            seen[want] += 1
            assert bool(spans.meet(_c(both[0]), _c(both[1]))) == want, both
            assert bool(spans.meet(_c(both[1]), _c(both[0]))) == want, both
    assert min(seen.values()) > 500


def test_strided_rows_of_the_largest_sizes(spans):
    big = 2 ** 31 - 1
    assert spans.nested(_c([4096, 2 ** 30, big, 2 ** 42, 1, 0, 1, 0]))
    assert not spans.nested(_c([4096, 16, big, 2 ** 40, big, 2 ** 60, 1, 0]))  # sums that do not fit count as the largest
    assert not spans.nested(_c([4096, 16, 5, 0, 1, 0, 1, 0]))
    # keys and values of one buffer, entry by entry: [batch, entry, 2, head, 64 bytes]
    key = [4096, 64, 1000, 2 ** 31, 1 << 20, 2048, 16, 64]
    assert not spans.meet(_c(key), _c([4096 + 1024] + key[1:]))
    assert spans.meet(_c(key), _c([4096 + 1023] + key[1:]))


def _select(score=MB, sstride=16, groups=2, length=16, lengths=None, first=0, recent=0, budget=8, keep=2 * MB, kstride=8, kept=3 * MB,
            drop=None, dstride=0, ws=None, size=0):
    return _capi.lib().gsx_b200_budget_select(score, sstride, groups, length, lengths, first, recent, budget, keep, kstride,
                                              kept, drop, dstride, ws, size, None)


LONG = dict(length=400_000, sstride=400_000, score=64 * MB, ws=8 * MB, size=1 << 40)
SELECT = [dict(kept=2 * MB + 60), dict(kept=2 * MB - 4), dict(keep=MB + 124), dict(keep=MB), dict(kept=MB + 8), dict(lengths=3 * MB),
          dict(lengths=3 * MB + 4), dict(lengths=2 * MB + 4), dict(drop=2 * MB, dstride=16), dict(drop=2 * MB - 64, dstride=16),
          dict(drop=MB + 4, dstride=16), dict(drop=3 * MB + 4, dstride=16), dict(drop=4 * MB, dstride=16, lengths=4 * MB + 92),
          dict(keep=2 * MB, kstride=32, drop=2 * MB + 28, dstride=32),
          dict(LONG, ws=64 * MB), dict(LONG, keep=8 * MB), dict(LONG, kept=8 * MB + 64), dict(LONG, lengths=8 * MB),
          dict(LONG, drop=8 * MB, dstride=400_000)]


@pytest.mark.parametrize("kw", SELECT)
def test_select_refuses_overlaps(kw):
    assert _select(**kw) == gb.INVALID_ARGUMENT
    assert b"overlap" in _capi.lib().gsx_b200_last_error()


@pytest.mark.parametrize("kw", [dict(sstride=2 ** 41), dict(kstride=2 ** 41), dict(drop=5 * MB, dstride=2 ** 41)])
def test_select_refuses_strides_out_of_range(kw):
    assert _select(**kw) == gb.OUT_OF_RANGE


def _gather(*fields, outer=1, inner=1, length=16, budget=8, keep=MB, kstride=8, kept=2 * MB, bad=None):
    base = dict(src=64 * MB, dst=4 * MB, row_bytes=12, src_row_stride=12, dst_row_stride=12)
    table = (_capi.GatherField * len(fields))(*[_capi.GatherField(**dict(base, **f)) for f in fields])
    return _capi.lib().gsx_b200_budget_gather(table, len(fields), outer, inner, length, budget, keep, kstride, kept, bad, None)


GATHER = [([{}, {}], {}), ([{}, dict(dst=4 * MB + 92)], {}), ([{}, dict(dst=4 * MB - 92)], {}),
          ([dict(dst_inner_stride=0)], dict(inner=2)), ([dict(dst_inner_stride=84)], dict(inner=2)),
          ([dict(dst_outer_stride=0, dst_inner_stride=96)], dict(outer=2, inner=3)),
          ([dict(dst_outer_stride=200, dst_inner_stride=96)], dict(outer=2, inner=3)),
          ([dict(dst_row_stride=24, dst_inner_stride=8)], dict(inner=2)),
          ([dict(dst=MB + 28)], {}), ([dict(dst=MB - 92)], {}), ([dict(dst=2 * MB)], {}), ([dict(dst=2 * MB - 92)], {}),
          ([dict(dst=5 * MB - 92)], dict(bad=5 * MB)), ([{}], dict(inner=2, keep=4 * MB + 100)),
          ([dict(dst_row_stride=32), dict(dst=4 * MB + 8, dst_row_stride=32)], {}),
          ([dict(dst_row_stride=32), dict(dst=4 * MB + 224 + 8, dst_row_stride=24)], {})]


@pytest.mark.parametrize("fields,kw", GATHER)
def test_gather_refuses_overlaps(fields, kw):
    inner = kw.get("inner", 1)
    fields = [dict(dict(dst_inner_stride=96) if inner > 1 else {}, **f) for f in fields]
    assert _gather(*fields, **kw) == gb.INVALID_ARGUMENT
    assert b"overlap" in _capi.lib().gsx_b200_last_error()


def test_gather_refuses_strides_out_of_range():
    assert _gather(dict(dst_inner_stride=96), inner=2, kstride=2 ** 41) == gb.OUT_OF_RANGE


def _accumulate(score=MB, weights=64 * MB, groups=3, rows=2, length=16, stride=16, lengths=None, row_lengths=None, out=2 * MB):
    return _capi.lib().gsx_b200_budget_accumulate(score, stride, weights, 0, 32, 16, groups, rows, length, lengths, row_lengths,
                                                  1.0, out, stride, None)


@pytest.mark.parametrize("kw", [dict(lengths=2 * MB), dict(row_lengths=2 * MB + 188), dict(lengths=2 * MB - 8),
                                dict(row_lengths=2 * MB + 124, stride=32), dict(out=MB, lengths=MB + 64)])
def test_accumulate_refuses_an_out_over_the_lengths(kw):
    assert _accumulate(**kw) == gb.INVALID_ARGUMENT
    assert b"overlap" in _capi.lib().gsx_b200_last_error()


def _backward(grad=64 * MB, index=32 * MB, itype=13, count=20, table=MB, rows=4, dim=8, stride=8, ws=8 * MB):
    L = _capi.lib()
    return L.gsx_b200_embedding_backward(grad, 0, stride, index, itype, count, 1.0, -1, table, 0, rows, dim, stride, 0, ws,
                                         L.gsx_b200_embedding_workspace_bytes(count, rows, dim), None, None)


@pytest.mark.parametrize("kw", [dict(ws=MB), dict(ws=MB + 112), dict(ws=MB - 256), dict(ws=64 * MB + 624), dict(ws=64 * MB - 16),
                                dict(ws=32 * MB + 144), dict(ws=32 * MB - 256), dict(ws=MB, rows=5000, count=9000),
                                dict(ws=32 * MB + 35_984, itype=12, rows=5000, count=9000)])
def test_backward_refuses_a_workspace_over_its_operands(kw):
    assert _backward(**kw) == gb.INVALID_ARGUMENT
    assert b"overlap" in _capi.lib().gsx_b200_last_error()


def test_a_flag_that_is_not_aligned_is_refused():
    """The kernels exchange it as one 32-bit word."""
    L = _capi.lib()
    bad = 128 * MB + 2
    assert L.gsx_b200_embedding_lookup(MB, 0, 4, 8, 8, 2 * MB, 12, 3, 1.0, 3 * MB, 0, 8, bad, None) == gb.INVALID_ARGUMENT
    assert L.gsx_b200_embedding_backward(MB, 0, 8, 2 * MB, 12, 3, 1.0, -1, 3 * MB, 0, 4, 8, 8, 0, 8 * MB, 1 << 40, bad,
                                         None) == gb.INVALID_ARGUMENT
    assert _gather({}, bad=bad) == gb.INVALID_ARGUMENT
