"""Accumulated weights, selection within a budget and the gather of the kept rows against plain forms.

Tolerance of the sums: u = 2^-24 an operation; any order of adding n terms is off by at most (n - 1) u sum|terms| to
first order (1.01 covers the rest), the decayed score being one more term with one more product."""
import numpy as np
import pytest
import torch

import gsx_b200 as gb

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check_accumulate(out, score, weights, decay, lengths=None, row_lengths=None):
    G, L = score.shape
    n = torch.full((G,), L, device="cuda") if lengths is None else lengths.long().clamp(0, L)
    m = torch.full((G,), weights.shape[1], device="cuda") if row_lengths is None else row_lengths.long().clamp(0, weights.shape[1])
    rows = torch.arange(weights.shape[1], device="cuda")[None, :, None] < m[:, None, None]
    used = torch.arange(L, device="cuda") < n[:, None]
    w = torch.where(rows & used[:, None, :], weights.double(), 0.0)
    d = float(torch.tensor(decay, dtype=F32))
    old = score.double() * d if decay != 0 else torch.zeros_like(score, dtype=torch.float64)
    want = old + w.sum(1)
    bound = 1.01 * U * (m[:, None] + 2) * (w.abs().sum(1) + old.abs())
    assert torch.equal(out[~used].view(torch.int32), score[~used].view(torch.int32))
    assert bool(((out.double() - want).abs() <= bound)[used].all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("groups,rows,length", [(1, 0, 5), (1, 1, 1), (3, 1, 8), (2, 3, 1000), (5, 64, 257), (1, 200, 2048),
                                                (2, 130, 4099), (4, 1000, 64), (1, 5000, 1), (70, 8, 33), (1, 8, 100_000), (2, 40, 1004),
                                                (3, 6, 1002), (1, 70, 514), (2, 33, 1001), (1, 9, 3)])
def test_accumulate_sizes(cuda_device, groups, rows, length, dtype):
    g = _gen(groups * 7 + rows + length)
    score = torch.rand(groups, length, generator=g, device="cuda")
    weights = torch.rand(groups, rows, length, generator=g, device="cuda").to(dtype)
    for decay in (1.0, 0.9, 0.0):
        out = gb.budget_accumulate(score, weights, out=torch.empty_like(score), decay=decay)
        _check_accumulate(out, score, weights, decay)
    same = gb.budget_accumulate(score, weights, out=torch.empty_like(score), decay=0.0)
    assert torch.equal(out, same)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,length", [(4, 999), (100, 1024), (300, 500)])
def test_accumulate_ragged_reads_nothing_behind_the_ends(cuda_device, rows, length, dtype):
    g = _gen(rows)
    score = torch.rand(6, length, generator=g, device="cuda")
    weights = torch.rand(6, rows, length, generator=g, device="cuda").to(dtype)
    lengths = torch.tensor([0, 1, length // 2, length, length + 9, -4], dtype=torch.int32, device="cuda")
    row_lengths = torch.tensor([rows, 0, 1, rows // 2, rows + 3, rows], dtype=torch.int32, device="cuda")
    for i in range(6):
        weights[i, max(0, min(rows, int(row_lengths[i]))):] = float("nan")
        weights[i, :, max(0, min(length, int(lengths[i]))):] = float("inf")
        score[i, max(0, min(length, int(lengths[i]))):] = float("nan")
    out = gb.budget_accumulate(score, weights, out=torch.empty_like(score), decay=0.5, lengths=lengths, row_lengths=row_lengths)
    _check_accumulate(out, score, weights, 0.5, lengths, row_lengths)
    inplace = score.clone()
    assert gb.budget_accumulate(inplace, weights, decay=0.5, lengths=lengths, row_lengths=row_lengths) is inplace
    assert torch.equal(inplace.view(torch.int32), out.view(torch.int32))
    score[:] = float("nan")  # decay 0 does not read the scores in use
    out = gb.budget_accumulate(score, weights, out=torch.empty_like(score), decay=0.0, lengths=lengths, row_lengths=row_lengths)
    _check_accumulate(out, score, weights, 0.0, lengths, row_lengths)


def test_accumulate_strided_and_unaligned(cuda_device):
    g = _gen(3)
    big = torch.rand(2, 3, 40, 131, generator=g, device="cuda").to(F16)
    for lo, hi in [(0, 128), (1, 129), (8, 72), (3, 130)]:
        w = big[..., lo:hi]
        buf = torch.rand(2, 3, 200, generator=g, device="cuda")
        score = buf[..., 5:5 + hi - lo]
        out = gb.budget_accumulate(score, w, out=torch.empty(2, 3, hi - lo, device="cuda"), decay=0.75)
        _check_accumulate(out.view(6, -1), score.reshape(6, -1), w.reshape(6, 40, -1), 0.75)
    one = torch.rand(500, generator=g, device="cuda")
    out = gb.budget_accumulate(one, big[0, 0, :7, :100].repeat(1, 5))
    assert out is one


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("groups,rows,length", [(1, 32, 8), (3, 33, 7), (2, 40, 9), (5, 71, 247), (2, 64, 249), (1, 600, 1003), (2, 300, 251),
                                                (2, 37, 2050), (40, 35, 501)])
def test_accumulate_many_rows_that_start_anywhere(cuda_device, groups, rows, length, dtype):
    """Odd lengths, starts at every element of a 16-byte block, rows next to one another or apart, groups inside rows,
    and lengths that end inside a block; what lies outside the weights is NaN."""
    g = _gen(rows + length)
    score = torch.rand(groups, length, generator=g, device="cuda")
    lengths = torch.randint(0, length + 1, (groups,), generator=g, device="cuda", dtype=torch.int32)
    row_lengths = torch.randint(0, rows + 1, (groups,), generator=g, device="cuda", dtype=torch.int32)
    for start in (0, 1, 3, 6):
        for pad in (0, 1, 5):
            for inside in (False, True):
                shape = (rows, groups, length + pad) if inside else (groups, rows, length + pad)
                count = shape[0] * shape[1] * shape[2]
                buf = torch.full((start + count + 9,), float("nan"), device="cuda", dtype=dtype)
                w = buf[start:start + count].view(shape)[..., :length]
                w = w.transpose(0, 1) if inside else w
                w.copy_(torch.rand(groups, rows, length, generator=g, device="cuda"))
                out = gb.budget_accumulate(score, w, out=torch.empty_like(score), decay=0.5)
                _check_accumulate(out, score, w, 0.5)
                out = gb.budget_accumulate(score, w, out=torch.empty_like(score), decay=0.5, lengths=lengths, row_lengths=row_lengths)
                _check_accumulate(out, score, w, 0.5, lengths, row_lengths)
    alike = w[:1, :, :].expand(groups, rows, length)  # the same weights for all groups
    out = gb.budget_accumulate(score, alike, out=torch.empty_like(score), decay=0.5)
    _check_accumulate(out, score, alike, 0.5)


def test_accumulate_scores_at_every_alignment(cuda_device):
    g = _gen(9)
    for dtype in (F32, F16):
        for rows in (3, 40):
            w = torch.rand(3, rows, 64, generator=g, device="cuda").to(dtype)
            for a, b, step in [(0, 0, 64), (1, 0, 64), (0, 2, 64), (4, 4, 68), (0, 0, 65), (8, 3, 72)]:
                score = torch.rand(300, generator=g, device="cuda")[a:a + 3 * step].view(3, step)[:, :64]
                out = torch.full((300,), 7.0, device="cuda")
                to = out[b:b + 3 * step].view(3, step)[:, :64]
                gb.budget_accumulate(score, w, out=to, decay=0.25)
                _check_accumulate(to, score, w, 0.25)
                to.fill_(7.0)
                assert bool((out == 7.0).all())


def test_accumulate_offsets_behind_32_bits(cuda_device):
    """Weights of more than 2^32 elements (8.6 GB): the last group's rows are read from their own place."""
    G, R, L = 3, 1500, 1_000_000
    w = torch.zeros(G, R, L, dtype=F16, device="cuda")
    w[2, R - 1, L - 5:] = 3.0
    w[0, 7, 11] = 2.0
    score = torch.ones(G, L, device="cuda")
    out = gb.budget_accumulate(score, w, out=torch.empty_like(score), decay=1.0)
    want = torch.ones(G, L, device="cuda")
    want[2, L - 5:] = 4.0
    want[0, 11] = 3.0
    assert torch.equal(out, want)


def _plain_select(score, budget, n, first, recent):
    """One group in numpy: the kept and the dropped entries."""
    n = max(0, min(len(score), n))
    if n <= budget:
        return np.arange(n), np.arange(0)
    middle = np.arange(first, n - recent)
    s = score[middle].astype(np.float64)
    nan = np.isnan(s)
    order = np.lexsort((middle, -np.where(nan, 0.0, s), nan))  # NaN last, then the largest, then the lowest index
    best = middle[order][:budget - first - recent]
    keep = np.sort(np.concatenate([np.arange(first), best, np.arange(n - recent, n)]))
    return keep, np.setdiff1d(np.arange(n), keep)


def _check_select(score, budget, lengths=None, first=0, recent=0):
    G, L = score.shape
    keep = torch.full((G, max(budget, 1)), -7, dtype=torch.int32, device="cuda")
    kept = torch.full((G,), -7, dtype=torch.int32, device="cuda")
    drop = torch.full((G, L), -7, dtype=torch.int32, device="cuda")
    gb.budget_select(score, budget, lengths=lengths, first=first, recent=recent, keep=keep, kept=kept, drop=drop)
    keep2, kept2 = gb.budget_select(score, budget, lengths=lengths, first=first, recent=recent)
    s = score.cpu().numpy()
    keep, kept, drop, keep2 = keep.cpu().numpy(), kept.cpu().numpy(), drop.cpu().numpy(), keep2.cpu().numpy()
    assert kept.tolist() == kept2.reshape(-1).cpu().tolist()
    for g in range(G):
        want, rest = _plain_select(s[g], budget, L if lengths is None else int(lengths[g]), first, recent)
        assert kept[g] == len(want)
        assert np.array_equal(keep[g, :len(want)], want)
        assert (keep[g, len(want):] == -7).all()
        assert np.array_equal(drop[g, :len(rest)], rest)
        assert (drop[g, len(rest):] == -7).all()
        assert np.array_equal(keep2.reshape(G, -1)[g, :len(want)], want)


SELECT_SIZES = [(1, 1, 0), (1, 1, 1), (2, 5, 3), (3, 33, 32), (4, 1000, 1), (2, 1025, 1024), (3, 5000, 2500),
                (1, 49_152, 30_000), (2, 49_153, 100), (3, 100_001, 77_777), (1, 400_000, 399_999), (40, 60_000, 512), (3, 131_072, 20_000), (2, 131_073, 200),
                (2, 393_217, 200_000), (1, 1_000_003, 400_000), (5, 500_000, 7)]


@pytest.mark.parametrize("groups,length,budget", SELECT_SIZES)
def test_select_sizes(cuda_device, groups, length, budget):
    g = _gen(length + budget)
    score = torch.exp(2.0 * torch.randn(groups, length, generator=g, device="cuda"))
    _check_select(score, budget)
    first, recent = min(4, budget), (budget - min(4, budget)) // 3
    _check_select(score, budget, first=first, recent=recent)
    _check_select(score, budget, first=budget)  # only the first ones stay
    _check_select(score, budget, recent=budget)


@pytest.mark.parametrize("length", [2000, 60_000, 420_000])
def test_select_ties_and_special_values(cuda_device, length):
    g = _gen(length)
    base = torch.randint(0, 4, (1, length), generator=g, device="cuda").float()
    special = torch.randn(1, length, generator=g, device="cuda")
    pick = torch.randint(0, 8, (1, length), generator=g, device="cuda")
    for v, x in enumerate([float("nan"), float("inf"), float("-inf"), 0.0, -0.0, -1e-42, 3.4e38]):
        special = torch.where(pick == v, torch.tensor(x, device="cuda"), special)
    for score in (base, torch.zeros(1, length, device="cuda"), special, -special, torch.full((1, length), float("nan"), device="cuda")):
        for budget in (1, length // 7, length // 2, length - 1):
            _check_select(score, budget)
            _check_select(score, budget, first=budget // 5, recent=budget // 4)


@pytest.mark.parametrize("length", [300, 70_000, 400_000])
def test_select_ragged(cuda_device, length):
    g = _gen(5)
    score = torch.rand(7, length, generator=g, device="cuda")
    lengths = torch.tensor([0, 1, 5, length // 2, length, length + 5, -2], dtype=torch.int32, device="cuda")
    for i in range(7):
        score[i, max(0, min(length, int(lengths[i]))):] = float("inf")  # never chosen
    for budget in (5, length // 2, length, length + 100):
        _check_select(score, budget, lengths=lengths)
        _check_select(score, budget, lengths=lengths, first=2, recent=3)


def test_select_shapes_and_strides(cuda_device):
    g = _gen(6)
    wide = torch.rand(3, 4, 70, generator=g, device="cuda")
    keep, kept = gb.budget_select(wide[..., 1:61], 10, recent=2)
    assert keep.shape == (3, 4, 10) and kept.shape == (3, 4)
    for b in range(3):
        for h in range(4):
            assert np.array_equal(keep[b, h].cpu().numpy(), _plain_select(wide[b, h, 1:61].cpu().numpy(), 10, 60, 0, 2)[0])
    keep, kept = gb.budget_select(wide[0, 0], 9)
    assert keep.shape == (9,) and kept.shape == ()
    assert int(kept) == 9


@pytest.mark.parametrize("dtype,tail", [(F32, (3,)), (F32, ()), (torch.uint8, (5,)), (F16, (7,)), (F16, (128,)),
                                        (F32, (15, 3)), (torch.int64, (2,)), (torch.uint8, (20_001,)), (F32, (2,)),
                                        (F32, (4,)), (F32, (5,)), (F32, (6,)), (F32, (7,)), (F32, (8,)), (F32, (9,)),
                                        (F16, (6,)), (F16, (1,)), (torch.uint8, (1,)), (torch.int64, (1,))])
def test_gather_rows_of_every_size(cuda_device, dtype, tail):
    g = _gen(7)
    # lists that keep few entries and lists that keep most
    for rows, n in ((1000, 399), (6000, 2500), (5000, 1024), (7000, 5001), (4100, 4096), (9, 5), (300_000, 700)):
        src = torch.randint(0, 200, (rows, *tail), generator=g, device="cuda").to(dtype)
        keep = torch.sort(torch.randperm(rows, generator=g, device="cuda")[:n + 1]).values.int()
        kept = torch.tensor(n, dtype=torch.int32, device="cuda")
        if tail == (20_001,) and rows > 6000:
            continue
        for offset in (0, 1):  # a dst that starts on a 16-byte boundary, and one that need not
            dst = torch.full((n + 11, *tail), 77, device="cuda").to(dtype)
            gb.budget_gather([(src, dst[offset:])], keep, kept)
            assert torch.equal(dst[offset:offset + n], src[keep[:n].long()])
            assert bool((dst[offset + n:] == 77).all()) and bool((dst[:offset] == 77).all())


@pytest.mark.parametrize("dim", [1, 2, 3, 4])
def test_gather_short_rows_in_any_order_and_from_any_place(cuda_device, dim):
    """Lists need not be sorted, may name an entry twice, and src may be strided or start anywhere."""
    g = _gen(17)
    flat = torch.randn(5000 * dim + 8, generator=g, device="cuda")
    keep = torch.randint(1000, 2500, (3000,), generator=g, device="cuda", dtype=torch.int32)
    kept = torch.tensor(2999, dtype=torch.int32, device="cuda")
    for src in [flat[o:o + 5000 * dim].view(5000, dim) for o in range(4)] + [torch.randn(5000, dim + 1, generator=g, device="cuda")[:, :dim]]:
        dst = torch.zeros(3000, dim, device="cuda")
        gb.budget_gather([(src, dst)], keep, kept)
        assert torch.equal(dst[:2999], src[keep[:2999].long()]) and bool((dst[2999] == 0).all())
    one = torch.tensor([4999, 0], dtype=torch.int32, device="cuda")  # a single row, and the last word of src
    dst = torch.zeros(2, dim, device="cuda")
    gb.budget_gather([(flat[8:].view(5000, dim), dst)], one, torch.tensor(1, dtype=torch.int32, device="cuda"))
    assert torch.equal(dst[0], flat[8:].view(5000, dim)[4999])


@pytest.mark.parametrize("order", ["heads first", "entries first"])
def test_gather_caches_of_both_layouts(cuda_device, order):
    g = _gen(8)
    B, H, S, D, budget = 3, 5, 200, 40, 64
    score = torch.rand(B, H, S, generator=g, device="cuda")
    lengths = torch.randint(0, S + 1, (B, H), generator=g, device="cuda", dtype=torch.int32)
    def cache(n):
        if order == "heads first":
            return torch.randn(B, H, n, D, generator=g, device="cuda").to(BF16)
        return torch.randn(B, n, H, D, generator=g, device="cuda").to(BF16).transpose(1, 2)
    k, v, k2, v2 = cache(S), cache(S), cache(budget), cache(budget)
    s2 = torch.zeros(B, H, budget, device="cuda")
    k0 = k2.clone()
    keep, kept = gb.budget_select(score, budget, lengths=lengths, first=4, recent=16)
    gb.budget_gather([(k, k2), (v, v2), (score, s2)], keep, kept)
    for b in range(B):
        for h in range(H):
            n = int(kept[b, h])
            i = keep[b, h, :n].long()
            assert torch.equal(k2[b, h, :n], k[b, h, i]) and torch.equal(v2[b, h, :n], v[b, h, i])
            assert torch.equal(s2[b, h, :n], score[b, h, i])
            assert torch.equal(k2[b, h, n:], k0[b, h, n:])


def test_gather_offsets_behind_32_bits(cuda_device):
    for row in (12, 1008):  # short rows and long ones, 4.8 GB each
        n = 4_800_000_000 // row
        src = torch.zeros(n, row, dtype=torch.uint8, device="cuda")
        src[-1] = 9
        src[-3] = 4
        keep = torch.tensor([0, n - 3, n - 1], dtype=torch.int32, device="cuda")
        dst = torch.full((3, row), 1, dtype=torch.uint8, device="cuda")
        gb.budget_gather([(src, dst)], keep, torch.tensor(3, dtype=torch.int32, device="cuda"))
        assert dst[:, 0].tolist() == [0, 4, 9] and torch.equal(dst, dst[:, :1].expand(3, row))
        del src


@pytest.mark.parametrize("dim", [1, 3, 4, 9])
def test_gather_flags_entries_out_of_range(cuda_device, dim):
    src = torch.randn(10, dim, device="cuda")
    dst = torch.zeros(4, dim, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    keep = torch.tensor([1, 10, -1, 9], dtype=torch.int32, device="cuda")
    gb.budget_gather([(src, dst)], keep, torch.tensor(1, dtype=torch.int32, device="cuda"), bad=bad)
    assert int(bad) == 0
    gb.budget_gather([(src, dst)], keep, torch.tensor(9, dtype=torch.int32, device="cuda"), bad=bad)
    assert int(bad) == 1
    assert torch.equal(dst, torch.stack([src[1], src[0] * 0, src[0] * 0, src[9]]))


@pytest.mark.parametrize("length", [900, 80_000, 400_000])
def test_evict_on_another_stream_and_in_a_replayed_graph(cuda_device, length):
    g = _gen(9)
    budget = length // 2
    score = torch.rand(4, length, generator=g, device="cuda")
    weights = torch.rand(4, 8, length, generator=g, device="cuda")
    src = torch.randn(4, length, 16, generator=g, device="cuda")

    def step(out, dst, keep, kept, stream=None):
        gb.budget_accumulate(score, weights, out=out, decay=0.5, stream=stream)
        gb.budget_select(out, budget, recent=7, keep=keep, kept=kept, stream=stream)
        gb.budget_gather([(src, dst)], keep, kept, stream=stream)

    def buffers():
        return (torch.empty_like(score), torch.empty(4, budget, 16, device="cuda"),
                torch.empty(4, budget, dtype=torch.int32, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda"))

    a, b, c, d = buffers(), buffers(), buffers(), buffers()
    step(*a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    step(*b, stream=side)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph, out in zip(graphs, (c, d)):
        with torch.cuda.graph(graph):
            step(*out)
    score.mul_(-1.0)
    step(*a)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()  # two captured calls at once
    graphs[0].replay()
    with torch.cuda.stream(other):
        graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    assert all(torch.equal(x, y) for x, y in zip(a, d))


def test_refusals(cuda_device):
    score = torch.rand(3, 20, device="cuda")
    w = torch.rand(3, 2, 20, device="cuda")
    keep, kept = gb.budget_select(score, 5)

    def refused(code, f, *args, **kw):
        with pytest.raises(gb.GsxError) as e:
            f(*args, **kw)
        assert e.value.code == code, e.value

    bad = gb.INVALID_ARGUMENT
    refused(bad, gb.budget_accumulate, score.double(), w)
    refused(bad, gb.budget_accumulate, score, w[:2])
    refused(bad, gb.budget_accumulate, score, w[..., :19])
    refused(bad, gb.budget_accumulate, score, w.cpu())
    refused(bad, gb.budget_accumulate, score, w, out=torch.empty(3, 21, device="cuda"))
    refused(bad, gb.budget_accumulate, score, w, lengths=torch.zeros(3, device="cuda"))
    refused(bad, gb.budget_accumulate, score[:1].expand(3, 20), w)
    refused(bad, gb.budget_accumulate, w[:, 0], w)
    flat = torch.rand(63, device="cuda")
    refused(bad, gb.budget_accumulate, flat[:60].view(3, 20), w, out=flat[3:].view(3, 20))
    refused(gb.NOT_SUPPORTED, gb.budget_accumulate, score, w.double())
    refused(bad, gb.budget_select, score, 5, first=3, recent=3)
    refused(gb.OUT_OF_RANGE, gb.budget_select, score, -1)
    refused(gb.OUT_OF_RANGE, gb.budget_select, score, 5, first=-1)
    refused(bad, gb.budget_select, score, 5, keep=torch.empty(3, 4, dtype=torch.int32, device="cuda"))
    refused(bad, gb.budget_select, score, 5, keep=torch.empty(3, 5, device="cuda"))
    refused(bad, gb.budget_select, score.t(), 5)
    src, dst = torch.rand(3, 20, 4, device="cuda"), torch.rand(3, 5, 4, device="cuda")
    gb.budget_gather([(src, dst)], keep, kept)
    refused(bad, gb.budget_gather, [(src, dst[:, :4])], keep, kept)
    refused(bad, gb.budget_gather, [(src, dst), (src[:, :19], dst)], keep, kept)
    refused(bad, gb.budget_gather, [(src, src[:, :5])], keep, kept)
    refused(bad, gb.budget_gather, [(src, dst.transpose(1, 2).contiguous().transpose(1, 2))], keep, kept)
    refused(gb.NOT_SUPPORTED, gb.budget_gather, [(src, dst.half())], keep, kept)
    refused(gb.OUT_OF_RANGE, gb.budget_gather, [(src, dst)] * 33, keep, kept)
    refused(bad, gb.budget_gather, [(src, dst)], keep.long(), kept)


@pytest.mark.parametrize("kind", ["entry by entry", "head by head", "rows of two sizes"])
def test_gather_into_one_interleaved_buffer(cuda_device, kind):
    """Keys and values that share a buffer: their spans overlap, their rows do not."""
    g = _gen(18)
    B, H, S, budget = 2, 3, 100, 40
    if kind == "entry by entry":
        buf = torch.full((B, budget + 1, 2, H, 64), 7.0, device="cuda")
        k2, v2 = buf[:, :, 0].transpose(1, 2), buf[:, :, 1].transpose(1, 2)
    elif kind == "head by head":
        buf = torch.full((B, H, 2 * budget + 3, 64), 7.0, device="cuda")
        k2, v2 = buf[:, :, :budget], buf[:, :, budget + 3:]
    else:
        buf = torch.full((B, H, budget * 80 + 5), 7.0, device="cuda")
        k2 = buf.as_strided((B, H, budget, 64), (H * (budget * 80 + 5), budget * 80 + 5, 64, 1), 0)
        v2 = buf.as_strided((B, H, budget, 16), (H * (budget * 80 + 5), budget * 80 + 5, 16, 1), budget * 64)
    k = torch.randn(B, H, S, k2.shape[-1], generator=g, device="cuda")
    v = torch.randn(B, H, S, v2.shape[-1], generator=g, device="cuda")
    keep, kept = gb.budget_select(torch.rand(B, H, S, generator=g, device="cuda"), budget)
    gb.budget_gather([(k, k2), (v, v2)], keep, kept)
    at = keep.long()[..., None]
    assert torch.equal(k2[:, :, :budget], torch.gather(k, 2, at.expand(-1, -1, -1, k.shape[-1])))
    assert torch.equal(v2[:, :, :budget], torch.gather(v, 2, at.expand(-1, -1, -1, v.shape[-1])))
    assert int((buf != 7.0).sum()) == k2[:, :, :budget].numel() + v2[:, :, :budget].numel()
    for bad in ([(k, k2), (k, k2)], [(k, k2[:, :1].expand(B, H, k2.shape[2], k2.shape[3]))]):
        with pytest.raises(gb.GsxError) as e:
            gb.budget_gather(bad, keep, kept)
        assert e.value.code == gb.INVALID_ARGUMENT
