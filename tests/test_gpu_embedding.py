"""Shared-row lookup and its gradient against the formulas in 64 bits.

Tolerances.  u = 2^-24 is the largest relative error of one f32 operation; a rounding to type t adds
finfo(t).eps / 2 relative, or half a step of its smallest subnormal.  Lookup: one product, one rounding.  Gradient:
any order of adding n terms is off by at most (n - 1) u sum|g| (to first order; 1.01 covers the rest), then one
product, with accumulate one fused product and sum, and one rounding."""
import pytest
import torch

import gsx_b200 as gb

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _half_step(dtype, exact):
    info = torch.finfo(dtype)
    return (exact.abs() * (info.eps / 2)).clamp_min(info.tiny * info.eps / 2)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _index(g, count, rows, dtype, skew=1.0):
    u = torch.rand(count, generator=g, device="cuda", dtype=torch.float64).pow(skew)
    return (u * rows).long().clamp_(max=rows - 1).to(dtype)


def _check_lookup(out, table, index, scale):
    want = table.double()[index.long()] * float(torch.tensor(scale, dtype=F32))
    bound = 1.01 * (want.abs() * U + _half_step(out.dtype, want))
    assert out.shape == want.shape
    assert bool(((out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
@pytest.mark.parametrize("out_type", [F32, F16, BF16])
@pytest.mark.parametrize("table_type", [F32, F16, BF16])
def test_lookup_types(cuda_device, table_type, out_type, itype):
    g = _gen(1)
    for count, rows, dim in [(1, 1, 1), (1, 5, 4096), (7, 3, 8), (1000, 17, 3), (1001, 300, 45), (513, 1000, 128),
                             (40, 2, 12), (4, 7, 2709), (43, 9, 685), (999, 20, 131), (130, 6, 33), (77, 9, 6),
                             (77, 9, 20), (50, 9, 300)]:
        table = torch.randn(rows, dim, generator=g, device="cuda").to(table_type)
        index = _index(g, count, rows, itype)
        _check_lookup(gb.embedding_lookup(table, index, out=torch.empty(count, dim, dtype=out_type, device="cuda"),
                                          scale=1.7), table, index, 1.7)


def test_lookup_large_takes_every_path(cuda_device):
    g = _gen(2)
    for count, rows, dim, dtype in [(400_003, 4096, 3, F32), (200_001, 1000, 45, BF16), (300_000, 64, 32, F16),
                                    (3_000_001, 1, 1, F32), (1_500_000, 700, 9, F16), (70_001, 5, 31, BF16),
                                    (100_003, 50, 130, BF16), (200_000, 40, 28, F16)]:
        table = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
        for itype in (torch.int32, torch.int64):
            index = _index(g, count, rows, itype, 2.0)
            _check_lookup(gb.embedding_lookup(table, index, scale=0.25), table, index, 0.25)
            index[5::7] = rows  # rows that stay as they were
            out, bad = torch.full((count, dim), 7.0, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
            gb.embedding_lookup(table, index, out=out, scale=0.25, bad=bad)
            assert int(bad) == 1 and bool((out[5::7] == 7.0).all())
            used = index < rows
            _check_lookup(out[used], table, index[used], 0.25)


def test_lookup_index_shapes_and_empty_calls(cuda_device):
    g = _gen(3)
    table = torch.randn(11, 6, generator=g, device="cuda")
    index = _index(g, 24, 11, torch.int64).view(2, 3, 4)
    out = gb.embedding_lookup(table, index)
    assert out.shape == (2, 3, 4, 6)
    assert torch.equal(out, table[index])
    assert gb.embedding_lookup(table, index[:0]).shape == (0, 3, 4, 6)
    assert gb.embedding_lookup(table[:, :0], index).shape == (2, 3, 4, 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lookup_strided_and_unaligned(cuda_device, dtype):
    g = _gen(4)
    wide = torch.randn(50, 83, generator=g, device="cuda").to(dtype)
    index = _index(g, 333, 50, torch.int32)
    for table in (wide[:, :16], wide[:, 1:17], wide[:, 2:47], wide.view(-1)[1:1 + 48 * 8].view(48, 8)[:, :8]):
        ix = index % table.shape[0]
        buf = torch.full((333, 100), 9.0, dtype=dtype, device="cuda")
        out = buf[:, 3:3 + table.shape[1]]
        gb.embedding_lookup(table, ix, out=out, scale=2.0)
        assert torch.equal(out, table[ix.long()] * 2.0)
        assert bool((buf[:, :3] == 9.0).all()) and bool((buf[:, 3 + table.shape[1]:] == 9.0).all())


@pytest.mark.parametrize("dim", [3, 8, 64])
def test_lookup_out_of_range_rows_are_left_and_flagged(cuda_device, dim):
    table = torch.randn(10, dim, device="cuda")
    index = torch.tensor([3, -1, 9, 10, 2 ** 40, 0], device="cuda")
    out = torch.full((6, dim), 5.0, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    gb.embedding_lookup(table, index[:1], out=out[:1], bad=bad)
    assert int(bad) == 0
    gb.embedding_lookup(table, index, out=out, bad=bad)
    assert int(bad) == 1
    assert bool((out[[1, 3, 4]] == 5.0).all())
    assert torch.equal(out[[0, 2, 5]], table[[3, 9, 0]])


def _check_gradient(got, grad, index, rows, scale, before=None, drop=None):
    index = index.reshape(-1).long()
    grad = grad.reshape(index.numel(), grad.shape[-1]).double()
    use = (index >= 0) & (index < rows)
    if drop is not None:
        use &= index != drop
    index, grad = index[use], grad[use]
    s = float(torch.tensor(scale, dtype=F32))
    want = torch.zeros(rows, grad.shape[1], dtype=torch.float64, device="cuda").index_add_(0, index, grad) * s
    size = torch.zeros_like(want).index_add_(0, index, grad.abs()) * abs(s)
    n = torch.bincount(index, minlength=rows).double()[:, None]
    bound = size * (n + 1) * U
    if before is not None:
        want = want + before.double()
        bound = bound + want.abs() * U
    bound = 1.01 * (bound + _half_step(got.dtype, want.abs() + bound))
    assert bool(((got.double() - want).abs() <= bound).all())
    if before is None:
        assert bool((got[(n == 0)[:, 0]] == 0).all())


GRADIENT_SIZES = [(0, 5, 3), (1, 1, 1), (5, 1, 4), (100, 256, 8), (8192, 300, 7), (8193, 300, 7), (5120, 70_000, 7), (5121, 70_000, 7), (148 * 1024 + 1, 300, 7), (30_000, 40_000, 130), (8192, 40_000, 900), (8193, 40_000, 900), (9000, 1, 3),
                  (20_000, 4096, 3), (20_000, 4097, 4), (50_000, 70_000, 2), (33_333, 5000, 45), (300, 1000, 2048),
                  (12_000, 3, 260), (2000, 50, 33), (200_001, 100, 1), (300_000, 1000, 2), (700_000, 4096, 3),
                  (150_000, 777, 4), (60_000, 1, 3), (700_001, 1000, 3), (1_300_000, 4096, 4),
                  (650_000, 17, 9), (620_000, 1152, 16), (606_208, 1, 1)]


@pytest.mark.parametrize("count,rows,dim", GRADIENT_SIZES)
def test_gradient_sizes(cuda_device, count, rows, dim):
    g = _gen(count + rows)
    grad = torch.randn(count, dim, generator=g, device="cuda")
    index = _index(g, count, rows, torch.int32, 2.0)
    got = gb.embedding_backward(grad, index, torch.full((rows, dim), float("nan"), device="cuda"), scale=0.3)
    _check_gradient(got, grad, index, rows, 0.3)
    again = gb.embedding_backward(grad, index, torch.empty(rows, dim, device="cuda"), scale=0.3)
    assert torch.equal(got, again)


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
@pytest.mark.parametrize("table_type", [F32, F16, BF16])
@pytest.mark.parametrize("grad_type", [F32, F16, BF16])
def test_gradient_types(cuda_device, grad_type, table_type, itype):
    g = _gen(5)
    for count, rows, dim in [(700, 40, 64), (9001, 600, 5), (900, 30, 16), (90_000, 300, 3), (80_000, 9, 1), (650_000, 300, 3)]:
        grad = torch.randn(count, dim, generator=g, device="cuda").to(grad_type)
        index = _index(g, count, rows, itype, 3.0)
        got = gb.embedding_backward(grad, index, torch.empty(rows, dim, dtype=table_type, device="cuda"), scale=1.5)
        _check_gradient(got, grad, index, rows, 1.5)
        before = torch.randn(rows, dim, generator=g, device="cuda").to(table_type)
        got = gb.embedding_backward(grad, index, before.clone(), scale=1.5, accumulate=True)
        _check_gradient(got, grad, index, rows, 1.5, before=before)


def test_gradient_three_digit_sort(cuda_device):
    rows = 2 ** 24 + 5
    g = _gen(6)
    grad = torch.randn(9000, 1, generator=g, device="cuda")
    index = _index(g, 9000, rows, torch.int64)
    index[:4000] = index[4000:8000]
    index[0], index[1] = rows - 1, 0
    got = gb.embedding_backward(grad, index, torch.empty(rows, 1, device="cuda"))
    _check_gradient(got, grad, index, rows, 1.0)


@pytest.mark.parametrize("count", [3000, 40_000, 300_000, 800_000])
@pytest.mark.parametrize("dim", [3, 64, 300])
def test_gradient_of_one_row_that_has_nearly_all(cuda_device, count, dim):
    g = _gen(7)
    grad = torch.randn(count, dim, generator=g, device="cuda")
    index = torch.full((count,), 4, dtype=torch.int32, device="cuda")
    index[::97] = _index(g, index[::97].numel(), 9, torch.int32)
    got = gb.embedding_backward(grad, index, torch.empty(9, dim, device="cuda"))
    _check_gradient(got, grad, index, 9, 1.0)


@pytest.mark.parametrize("dim", [3, 6])
@pytest.mark.parametrize("count,rows", [(500, 64), (500, 63), (30_000, 4096), (30_000, 9000), (90_000, 500), (800_000, 500)])
def test_gradient_drops_padding_and_out_of_range(cuda_device, count, rows, dim):
    g = _gen(8)
    grad = torch.randn(count, dim, generator=g, device="cuda")
    index = _index(g, count, rows, torch.int64)
    index[::5] = 7
    index[3::11] = rows + 2
    index[4::13] = -3
    used = (index != 7) & (index >= 0) & (index < rows)
    grad[~used] = float("nan")  # nothing of a dropped row may be seen
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = gb.embedding_backward(grad, index, torch.empty(rows, dim, device="cuda"), padding_row=7, bad=bad)
    assert int(bad) == 1
    _check_gradient(got, grad, index, rows, 1.0, drop=7)
    bad.zero_()
    fine = torch.where(used, index, 7)
    gb.embedding_backward(grad, fine, got, padding_row=7, bad=bad)
    assert int(bad) == 0
    _check_gradient(got, grad, fine, rows, 1.0, drop=7)
    none = torch.full_like(index, 7)
    assert bool((gb.embedding_backward(grad, none, got, padding_row=7) == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim,count", [(8, 10_000), (21, 10_000), (600, 10_000), (3, 100_000), (5, 800_000)])
def test_gradient_strided(cuda_device, dtype, dim, count):
    g = _gen(9)
    for offset in (0, 1):
        wide = torch.randn(count, dim + 8, generator=g, device="cuda").to(dtype)
        grad = wide[:, offset:offset + dim]
        index = _index(g, count, 77, torch.int32)
        buf = torch.full((77, dim + 16), 3.0, dtype=dtype, device="cuda")
        got = gb.embedding_backward(grad, index, buf[:, offset:offset + dim])
        _check_gradient(got, grad, index, 77, 1.0)
        rest = torch.cat([buf[:, :offset], buf[:, offset + dim:]], 1)
        assert bool((rest == 3.0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("count,rows,dim", [(500, 900, 4), (20_000, 3000, 40), (700_000, 2000, 3)])
def test_gradient_accumulated_leaves_unnamed_rows_to_the_bit(cuda_device, count, rows, dim, dtype):
    g = _gen(12)
    index = _index(g, count, rows // 2, torch.int32) * 2
    before = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    before[1::4] = -0.0
    before[3::8] = float("nan")
    before[7::16] = float("inf")
    got = gb.embedding_backward(torch.randn(count, dim, generator=g, device="cuda"), index, before.clone(), scale=-2.0,
                                accumulate=True)
    bits = torch.int32 if dtype == F32 else torch.int16
    assert torch.equal(got[1::2].view(bits), before[1::2].view(bits))
    assert not torch.equal(got[::2], before[::2])


def test_gradients_that_are_not_finite_stay_in_their_rows(cuda_device):
    for count, rows, dim in [(300, 20, 5), (50_000, 700, 24), (700_000, 300, 3)]:
        g = _gen(13)
        grad = torch.randn(count, dim, generator=g, device="cuda")
        index = _index(g, count, rows, torch.int64)
        grad[index == 3] = float("nan")
        grad[index == 5, 0] = float("inf")
        got = gb.embedding_backward(grad, index, torch.empty(rows, dim, device="cuda"))
        finite = torch.isfinite(got)
        assert not bool(finite[3].any()) and not bool(finite[5, 0])
        finite[3] = finite[5, 0] = True
        assert bool(finite.all())


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("dim", [1, 2, 3, 4, 5, 8, 9, 16, 17, 24, 33])
@pytest.mark.parametrize("count,rows", [(1, 1), (511, 3), (513, 300), (5000, 256), (5001, 257), (40_000, 500), (400_000, 40), (6000, 2600)])
def test_gradients_of_small_tables(cuda_device, count, rows, dim, dtype):
    """Tables that fit in shared memory: rows of every length, few rows (long lists) and many, popular rows, rows apart,
    a start at any element, padding and indices out of range."""
    g = _gen(count + dim)
    for pad, start in ((0, 0), (3, 1)):
        buf = torch.randn(count * (dim + pad) + start, generator=g, device="cuda").to(dtype)
        grad = buf[start:].view(count, dim + pad)[:, :dim]
        index = (torch.rand(count, generator=g, device="cuda").pow(2 + pad) * rows).int().clamp_(max=rows - 1)
        if count > 600:
            index[5] = -1
            index[600] = rows
        used = (index >= 0) & (index < rows)
        want = torch.zeros(rows, dim, dtype=torch.float64, device="cuda")
        want.index_add_(0, index[used].long(), grad[used].double())
        size = torch.zeros_like(want).index_add_(0, index[used].long(), grad[used].double().abs())
        n = torch.bincount(index[used].long(), minlength=rows).double()[:, None]
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = gb.embedding_backward(grad, index, torch.empty(rows, dim, device="cuda"), scale=0.75, bad=flag)
        assert bool(((got.double() - 0.75 * want).abs() <= 1.01 * U * 0.75 * size * (n + 2)).all())
        assert bool(flag.item()) == (count > 600)
        again = gb.embedding_backward(grad, index, torch.empty(rows, dim, device="cuda"), scale=0.75)
        assert torch.equal(got, again)


def test_offsets_behind_32_bits(cuda_device):
    """Tables, outputs and gradients of more than 4 GiB: their last rows are read and written at their own place."""
    dim = 1024
    rows = 2_300_000  # 4.7 GB of bf16
    index = torch.tensor([rows - 1, 5, rows - 2, rows - 1], device="cuda")
    table = torch.zeros(rows, dim, dtype=BF16, device="cuda")
    table[rows - 2:] = 3.0
    table[5] = 7.0
    out = gb.embedding_lookup(table, index, scale=2.0)
    assert out[:, 0].tolist() == [6.0, 14.0, 6.0, 6.0] and torch.equal(out, out[:, :1].expand(-1, dim))
    got = gb.embedding_backward(torch.ones(4, dim, dtype=BF16, device="cuda"), index, table)
    assert bool((got[rows - 1] == 2).all()) and bool((got[rows - 2] == 1).all()) and bool((got[5] == 1).all())
    assert int((got != 0).any(1).sum()) == 3
    del got
    grad = table.zero_()  # as a gradient of 2.3M positions
    grad[-1] = 4.0
    grad[1] = 0.5
    which = torch.zeros(rows, dtype=torch.int32, device="cuda")
    which[-1] = 1
    got = gb.embedding_backward(grad, which, torch.empty(300, dim, device="cuda"))
    assert bool((got[1] == 4).all()) and bool((got[0] == 0.5).all()) and bool((got[2:] == 0).all())
    small = torch.arange(12, device="cuda").view(3, 4).float()  # an out of more than 2^32 bytes, short rows
    where = torch.zeros(280_000_000, dtype=torch.int32, device="cuda")
    where[-1] = 2
    del table, grad, got
    out = gb.embedding_lookup(small, where)
    assert torch.equal(out[-1], small[2]) and torch.equal(out[-2], small[0]) and torch.equal(out[0], small[0])


def test_very_long_rows_and_empty_tables(cuda_device):
    g = _gen(14)
    for dim in (70_001, 65_536):
        table = torch.randn(3, dim, generator=g, device="cuda")
        index = torch.tensor([2, 0, 2, 1, 2], device="cuda")
        _check_lookup(gb.embedding_lookup(table, index, scale=3.0), table, index, 3.0)
        grad = torch.randn(5, dim, generator=g, device="cuda")
        _check_gradient(gb.embedding_backward(grad, index, torch.empty_like(table)), grad, index, 3, 1.0)
    for dim in (3, 8, 13):
        out, bad = torch.full((4, dim), 2.0, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        gb.embedding_lookup(torch.empty(0, dim, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), out=out, bad=bad)
        assert int(bad) == 1 and bool((out == 2.0).all())


def test_gradient_matches_differences_of_the_lookup(cuda_device):
    """A loss sum(c * lookup(table)) is linear in the table: moving one element by 1 moves it by its gradient."""
    g = _gen(10)
    table = torch.randint(-8, 9, (13, 5), generator=g, device="cuda").float()
    index = _index(g, 200, 13, torch.int32)
    c = torch.randint(-4, 5, (200, 5), generator=g, device="cuda").float()  # whole numbers: every sum is exact
    grad = gb.embedding_backward(c, index, torch.empty(13, 5, device="cuda"), scale=2.0)
    loss = lambda t: float((c * gb.embedding_lookup(t, index, scale=2.0)).double().sum())  # noqa: E731
    for v, k in [(0, 0), (5, 3), (12, 4)]:
        moved = table.clone()
        moved[v, k] += 1.0
        assert loss(moved) - loss(table) == float(grad[v, k])


def test_calls_on_another_stream_and_in_a_replayed_graph(cuda_device):
    g = _gen(11)
    table = torch.randn(500, 24, generator=g, device="cuda")
    index = _index(g, 20_000, 500, torch.int32)
    want_out = gb.embedding_lookup(table, index, scale=0.5)
    want = gb.embedding_backward(want_out, index, torch.empty_like(table))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = gb.embedding_lookup(table, index, scale=0.5, stream=side)
    got = gb.embedding_backward(out, index, torch.empty_like(table), stream=side)
    side.synchronize()
    assert torch.equal(out, want_out) and torch.equal(got, want)
    out, got = torch.zeros_like(out), torch.zeros_like(table)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gb.embedding_lookup(table, index, out=out, scale=0.5)
        gb.embedding_backward(out, index, got)
    gb.embedding_backward(want_out, index.flip(0).contiguous(), torch.empty_like(table))  # other work between
    table.add_(1.0)
    index.copy_(index.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    again = gb.embedding_lookup(table, index, scale=0.5)
    assert torch.equal(out, again)
    assert torch.equal(got, gb.embedding_backward(again, index, torch.empty_like(table)))


def test_refusals(cuda_device):
    table = torch.randn(10, 4, device="cuda")
    index = torch.zeros(6, dtype=torch.int32, device="cuda")
    grad = torch.zeros(6, 4, device="cuda")

    def refused(code, f, *args, **kw):
        with pytest.raises(gb.GsxError) as e:
            f(*args, **kw)
        assert e.value.code == code, e.value

    refused(gb.INVALID_ARGUMENT, gb.embedding_lookup, table[0], index)
    refused(gb.INVALID_ARGUMENT, gb.embedding_lookup, table, index.cpu())
    refused(gb.INVALID_ARGUMENT, gb.embedding_lookup, table, index, out=torch.empty(6, 5, device="cuda"))
    refused(gb.INVALID_ARGUMENT, gb.embedding_lookup, table.t(), index)
    refused(gb.INVALID_ARGUMENT, gb.embedding_lookup, table, index.repeat(2)[::2])
    refused(gb.NOT_SUPPORTED, gb.embedding_lookup, table.double(), index)
    refused(gb.NOT_SUPPORTED, gb.embedding_lookup, table, index.to(torch.int16))
    refused(gb.INVALID_ARGUMENT, gb.embedding_lookup, table, index, bad=torch.zeros(2, device="cuda"))
    refused(gb.INVALID_ARGUMENT, gb.embedding_backward, grad[:5], index, table)
    refused(gb.INVALID_ARGUMENT, gb.embedding_backward, grad[:1].expand(6, 4), index, table)
    refused(gb.INVALID_ARGUMENT, gb.embedding_backward, grad, index, table[:1].expand(10, 4))
    refused(gb.OUT_OF_RANGE, gb.embedding_backward, grad, index, table, padding_row=10)
    refused(gb.NOT_SUPPORTED, gb.embedding_backward, grad.double(), index, table)


def _check_whole(got, grad, index, rows, scale=1.0, before=None):
    """Whole numbers (and a scale that is a power of two): every sum below 2^24 is exact in any order, so the result is
    the formula's to the bit, however many positions a row has."""
    use = (index >= 0) & (index < rows)
    want = torch.zeros(rows, grad.shape[1], dtype=torch.float64, device="cuda").index_add_(0, index[use].long(), grad[use].double())
    assert float(torch.zeros_like(want).index_add_(0, index[use].long(), grad[use].double().abs()).max()) < 2 ** 24
    want = want * scale + (0 if before is None else before.double())
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("grad_type", [F32, BF16])
@pytest.mark.parametrize("count,rows,dim", GRADIENT_SIZES)
def test_gradient_sums_of_whole_numbers_are_exact(cuda_device, count, rows, dim, grad_type):
    """No part of a long row is lost or added twice: the bound of a sum of n rounded terms grows with n and would not see
    it."""
    g = _gen(count + rows + 1)
    grad = torch.randint(-4, 5, (count, dim), generator=g, device="cuda").to(grad_type)
    index = _index(g, count, rows, torch.int64, 2.0)
    index[3::101] = -1
    got = gb.embedding_backward(grad, index, torch.empty(rows, dim, device="cuda"), scale=0.5)
    _check_whole(got, grad, index, rows, 0.5)
    before = torch.randint(-9, 10, (rows, dim), generator=g, device="cuda").float()
    got = gb.embedding_backward(grad, index, before.clone(), scale=-2.0, accumulate=True)
    _check_whole(got, grad, index, rows, -2.0, before)


@pytest.mark.parametrize("start", [0, 1])
@pytest.mark.parametrize("count", [3000, 40_000, 300_000, 800_000])
@pytest.mark.parametrize("dim", [3, 64, 300])
def test_whole_sums_of_one_row_that_has_nearly_all(cuda_device, count, dim, start):
    g = _gen(15)
    grad = torch.randint(1, 5, (count * dim + start,), generator=g, device="cuda").float()[start:].view(count, dim)
    index = torch.full((count,), 4, dtype=torch.int32, device="cuda")
    index[::97] = _index(g, index[::97].numel(), 9, torch.int32)
    _check_whole(gb.embedding_backward(grad, index, torch.empty(9, dim, device="cuda")), grad, index, 9)
    wide = torch.empty(30_000, dim, device="cuda")  # a table of its own size: the sort of all positions
    _check_whole(gb.embedding_backward(grad, index, wide), grad, index, 30_000)
