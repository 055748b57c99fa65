"""The paged KV cache's operators on the GPU against a 64-bit restatement on
the host: lengths from none to several chunks, every head size, page size and
page type, shared heads, strided inputs, garbage in every place that no call may
read, and the calls as a cache makes them."""

import math

import pytest
import torch

from tests import paged_reference as R

pytestmark = pytest.mark.gpu

D16 = torch.float16


def kernels():
    from apple_amd import kernels as K

    return K


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32).to(device)


def poison(pool, table, lens):
    """NaN in every row that no sequence holds: behind the lengths, and in the pages that no table has."""
    held = torch.zeros((pool.count, pool.size), dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(n):
            page = int(table[b, i // pool.size])
            if 0 <= page < pool.count:
                held[page, i % pool.size] = True
    for name in ("k", "v"):
        if pool.kind == "fp16":
            getattr(pool, name)[(~held)[:, None, :].expand(-1, pool.heads, -1)] = math.nan
        else:
            getattr(pool, name + "_scale")[(~held)[:, None, :].expand(-1, pool.heads, -1)] = math.nan
    return pool


def same(got, want):
    """Equal values, NaN included."""
    return bool(((got.cpu().float() == want.float()) | (torch.isnan(got.cpu().float()) & torch.isnan(want.float()))).all())


def attend(device, pool, table, lens, q, scale, chosen=None):
    K = kernels()
    return K.paged_attention(q.to(device), pool.pages(device), table.to(device), i32(lens, device), scale,
                             None if chosen is None else chosen.to(device))


# ------------------------------------------------------------------ append, read

@pytest.mark.parametrize("kind", ["fp16", "int8", "e4m3"])
@pytest.mark.parametrize("dim, heads, size, starts, counts, pad", [
    (64, 8, 16, [0], [1], 0), (64, 2, 16, [15, 16, 0, 31], [1, 1, 1, 1], 0), (64, 5, 32, [3, 0, 40], [70, 0, 9], 5),
    (128, 3, 64, [0, 63, 64], [64, 2, 200], 3), (256, 1, 16, [7, 0], [33, 1], 0), (256, 6, 256, [250], [300], 1),
    (128, 4, 128, [0, 0, 0, 100], [0, 0, 0, 29], 9), (64, 1, 16, [0], [1000], 0)])
def test_append_and_read(device, kind, dim, heads, size, starts, counts, pad):
    K = kernels()
    ends = [a + n for a, n in zip(starts, counts)]
    pool = R.Pool(kind, sum(-(-e // size) for e in ends) + 2, heads, size, dim, seed=dim + size)
    table = pool.tables(ends)
    n = sum(counts)
    k, v = pool.randn((n + pad, heads, dim), 3.0), pool.randn((n + pad, heads, dim))
    k[0, 0] = 0
    pages = pool.pages(device)
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    one = all(c == 1 for c in counts) and not pad
    # strided rows, as of a fused projection's output
    wide = torch.zeros((n + pad, 2, heads, dim), dtype=D16, device=device)
    wide[:, 0], wide[:, 1] = k.to(device), v.to(device)
    K.paged_append(pages, table.to(device), i32(starts, device), wide[:, 0], wide[:, 1],
                   None if one else i32(cu, device))
    pool.append(table, starts, k, v, cu)
    for name, got in pages._asdict().items():
        want = getattr(pool, name)
        if want is not None:
            assert same(got, want), name
    # back: the appended range, and each sequence from its start
    for begin in (starts, [0] * len(starts)):
        m = [e - a for a, e in zip(begin, ends)]
        at = [0]
        for c in m:
            at.append(at[-1] + c)
        ko, vo = K.paged_read(pages, table.to(device), i32(begin, device), i32(at, device), at[-1] + 2)
        for b in range(len(starts)):
            wk, wv, _ = pool.window(table, b, begin[b], ends[b])
            # one fp32 product and one rounding, which 64 bits give as well but for values next to a border
            for got, want in ((ko, wk), (vo, wv)):
                got = got[at[b]:at[b + 1]].cpu().double()
                assert ((got - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -24) + 2.0 ** -25).all()
        assert not ko[at[-1]:].any() and not vo[at[-1]:].any()
        out = (torch.full_like(ko, 7.0), torch.full_like(vo, 8.0))
        K.paged_read(pages, table.to(device), i32(begin, device), i32(at, device), at[-1] + 2, out)
        assert torch.equal(out[0][:at[-1]], ko[:at[-1]]) and (out[0][at[-1]:] == 7.0).all() and (out[1][at[-1]:] == 8.0).all()


@pytest.mark.parametrize("batch", [63, 64, 200])
def test_append_and_read_of_many_sequences(device, batch):
    """More sequences than a wave's lanes hold, most of them with few rows or none, rows of one sequence in every wave."""
    K = kernels()
    g = torch.Generator().manual_seed(batch)
    starts = torch.randint(0, 40, (batch,), generator=g).tolist()
    counts = torch.randint(0, 5, (batch,), generator=g).tolist()
    counts[0], counts[batch // 2], counts[-1] = 0, 90, 3
    ends = [a + n for a, n in zip(starts, counts)]
    pool = R.Pool("int8", sum(-(-e // 16) for e in ends) + 1, 2, 16, 64, seed=batch)
    table, n = pool.tables(ends), sum(counts)
    k, v = pool.randn((n + 7, 2, 64)), pool.randn((n + 7, 2, 64))
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    pages = pool.pages(device)
    K.paged_append(pages, table.to(device), i32(starts, device), k.to(device), v.to(device), i32(cu, device))
    pool.append(table, starts, k, v, cu)
    for name, got in pages._asdict().items():
        assert same(got, getattr(pool, name)), name
    ko, vo = K.paged_read(pages, table.to(device), i32(starts, device), i32(cu, device), n + 7)
    for b in range(batch):
        wk, wv, _ = pool.window(table, b, starts[b], ends[b])
        for got, want in ((ko, wk), (vo, wv)):
            assert ((got[cu[b]:cu[b + 1]].cpu().double() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -24)).all()
    assert not ko[n:].any()


def test_no_sequences(device):
    """An empty batch: no rows, and zeros read back."""
    K = kernels()
    pages = R.Pool("fp16", 2, 2, 16, 64, seed=1).pages(device)
    table, lens, cu = torch.zeros((0, 3), dtype=torch.int32, device=device), i32([], device), i32([0], device)
    K.paged_append(pages, table, lens, *(torch.ones((5, 2, 64), dtype=D16, device=device),) * 2, cu)
    ko, vo = K.paged_read(pages, table, lens, cu, 5)
    assert not ko.any() and not vo.any()
    q = torch.ones((0, 4, 64), dtype=D16, device=device)
    assert K.paged_attention(q, pages, table, lens, 0.1).shape == (0, 4, 64)
    assert K.page_select(q, pages, table, lens, 3).shape == (0, 2, 3)
    # and sequences whose table has no columns
    table, lens, q = torch.zeros((2, 0), dtype=torch.int32, device=device), i32([4, 0], device), torch.ones((2, 4, 64), dtype=D16, device=device)
    assert not K.paged_attention(q, pages, table, lens, 0.1).any()
    assert (K.page_select(q, pages, table, lens, 3) == -1).all()


@pytest.mark.parametrize("kind", ["fp16", "int8", "e4m3"])
def test_rows_that_are_not_finite(device, kind):
    """A row with an infinity or NaN: as it is in fp16, scale NaN in 8 bits; bounds keep the NaN, later rows do not clear it."""
    K = kernels()
    pool = R.Pool(kind, 3, 2, 16, 64, seed=5)
    k, v = pool.randn((6, 2, 64)), pool.randn((6, 2, 64))
    k[1, 0, 3], k[2, 1, 5], v[3, 0, 9], v[4, 1, 1] = math.inf, math.nan, -math.inf, math.nan
    k[5, 1] *= 60000 / k[5, 1].abs().amax().float()  # near fp16's largest
    v[0, 1] = 6e-8                                   # and its smallest
    table, cu = torch.tensor([[1, 2]], dtype=torch.int32), [0, 6]
    pages = pool.pages(device)
    K.paged_append(pages, table.to(device), i32([12], device), k.to(device), v.to(device), i32(cu, device))
    pool.append(table, [12], k, v, cu)
    for name, got in pages._asdict().items():
        want = getattr(pool, name)
        if want is not None:
            assert same(got, want), name
    # row 2 went to position 14, in page 1: position 15 after it widens the same bounds
    K.paged_append(pages, table.to(device), i32([15], device), k[:1].to(device), v[:1].to(device))
    assert torch.isnan(pages.bounds[1, 1, :, 5]).all()


def test_pages_outside_the_pool_and_rows_past_the_table(device):
    """Entries that are no page, lengths past the table, a cu that is no prefix: nothing is written or read outside."""
    K = kernels()
    for kind in ("fp16", "int8"):
        pool = R.Pool(kind, 4, 2, 16, 64, seed=6)
        table = torch.tensor([[0, -1, 2], [99, 3, -7], [1, 4, 2147483647]], dtype=torch.int32)
        starts, counts = [10, 14, 30], [30, 20, 40]
        cu = [0, 30, 50, 90]
        k, v = pool.randn((90, 2, 64)), pool.randn((90, 2, 64))
        pages = pool.pages(device)
        K.paged_append(pages, table.to(device), i32(starts, device), k.to(device), v.to(device), i32(cu, device))
        pool.append(table, starts, k, v, cu)
        for name, got in pages._asdict().items():
            if getattr(pool, name) is not None:
                assert same(got, getattr(pool, name)), name
        ko, _ = K.paged_read(pages, table.to(device), i32(starts, device), i32(cu, device), 90)
        for b in range(3):
            want, _, there = pool.window(table, b, starts[b], starts[b] + counts[b])
            assert not ko[cu[b]:cu[b + 1]][(~there).to(device)].any()
            got = ko[cu[b]:cu[b + 1]].cpu().double()
            assert ((got - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -24)).all()
        before = [t.clone() for t in pages if t is not None]
        for bad in ([5, 5, 5, 5], [90, 60, 30, 0], [-4, 400, -4, 400], [100, 100, 100, 100]):
            K.paged_append(pages, table.to(device), i32([2147483647, -5, 47], device), k.to(device), v.to(device),
                           i32(bad, device))
            K.paged_read(pages, table.to(device), i32([2147483647, -5, 47], device), i32(bad, device), 90)
        q = torch.randn((3, 4, 64)).half()
        for lens in ([2147483647, -5, 48], [40, 33, 48]):
            got = attend(device, pool, table, lens, q, 0.125)
            R.check(got, *R.attention(pool, table, lens, q, 0.125), str(lens))
        torch.cuda.synchronize()
        assert len(before) == len([t for t in pages if t is not None])


@pytest.mark.parametrize("kind", ["fp16", "int8", "e4m3"])
@pytest.mark.parametrize("batch", [3, 70])
def test_row_offsets_that_are_no_prefix_write_nothing(device, kind, batch):
    """``cu`` that no row n has a sequence in (cu[b] <= n < cu[b + 1]): the pool stays as it is, and zeros are read."""
    K = kernels()
    pool = R.Pool(kind, 2 * batch, 2, 16, 64, seed=batch)
    table = torch.randperm(2 * batch, generator=pool.g).int().view(batch, 2).to(device)
    k, v = (pool.randn((90, 2, 64)).to(device) for _ in range(2))
    falling = [90 - 90 * i // batch for i in range(batch + 1)]
    for cu in ([5] * (batch + 1), falling, [100] * (batch + 1), [-7] * (batch + 1), [100 + i for i in range(batch + 1)],
               [-100 + i for i in range(batch + 1)]):
        for starts in ([0] * batch, [2147483647, -5, 31] + [9] * (batch - 3)):
            pages = pool.pages(device)
            K.paged_append(pages, table, i32(starts, device), k, v, i32(cu, device))
            for name, got in pages._asdict().items():
                want = getattr(pool, name)
                if want is not None:
                    assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8)), (name, cu[:4])
            for x in K.paged_read(pages, table, i32(starts, device), i32(cu, device), 90):
                assert not x.any(), cu[:4]
            out = tuple(torch.full((90, 2, 64), 3.0, dtype=D16, device=device) for _ in range(2))
            K.paged_read(pages, table, i32(starts, device), i32(cu, device), 90, out)
            assert (out[0] == 3.0).all() and (out[1] == 3.0).all()


@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("batch", [5, 63, 64, 130])
def test_any_row_offsets_stay_in_the_tables_pages(device, kind, batch):
    """``cu`` of any numbers and lengths past every table: only pages that a table names are written."""
    K = kernels()
    pool = R.Pool(kind, 3 * batch + 40, 2, 16, 64, seed=batch)
    order = torch.randperm(pool.count, generator=pool.g).int()
    table, rest = order[:2 * batch].view(batch, 2).clone(), order[2 * batch:].long()
    table[1, 0], table[2, 1] = -1, pool.count
    k, v = (pool.randn((300, 2, 64)).to(device) for _ in range(2))
    pages = pool.pages(device)
    for trial in range(12):
        cu = torch.randint(-50, 400, (batch + 1,), generator=pool.g, dtype=torch.int32)
        if trial % 3 == 0:
            cu[::2], cu[1::2] = -4, 300 + trial
        starts = torch.randint(-5, 60, (batch,), generator=pool.g, dtype=torch.int32)
        starts[trial % batch] = 2147483647
        K.paged_append(pages, table.to(device), starts.to(device), k, v, cu.to(device))
        for name, got in pages._asdict().items():
            want = getattr(pool, name)
            if want is not None:
                assert torch.equal(got.cpu()[rest].view(torch.uint8), want[rest].view(torch.uint8)), (name, trial)


# ------------------------------------------------------------------ attention

LENGTHS = [[0], [1], [15, 16, 17], [31, 0, 33, 64], [129, 1, 500, 511], [513, 2, 1200], [3001]]


@pytest.mark.parametrize("kind", ["fp16", "int8", "e4m3"])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
@pytest.mark.parametrize("dim, heads, group, size", [(64, 8, 4, 16), (64, 2, 1, 64), (128, 3, 8, 32), (128, 1, 16, 128),
                                                     (256, 2, 3, 16), (64, 1, 20, 256)])
def test_attention(device, kind, lens, dim, heads, group, size):
    pool = R.Pool(kind, sum(-(-n // size) for n in lens) + 2, heads, size, dim, seed=len(lens) + dim, bounds=False)
    table = pool.tables(lens)
    poison(pool, table, lens)
    q = pool.randn((len(lens), heads * group, dim), 2.0)
    got = attend(device, pool, table, lens, q, dim ** -0.5)
    R.check(got, *R.attention(pool, table, lens, q, dim ** -0.5))


@pytest.mark.parametrize("kind", ["fp16", "int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch", [4, 12])
def test_tables_far_wider_than_the_sequences(device, kind, dim, batch):
    """A table for 40,000 positions a sequence, as a captured step keeps: cut by the lengths on the device, in
    chunks and rows of few and of many."""
    lens = ([2100, 0, 33, 700] * 3)[:batch]
    pool = R.Pool(kind, sum(-(-n // 16) for n in lens) + 1, 8, 16, dim, seed=dim + batch, bounds=False)
    narrow = pool.tables(lens)
    poison(pool, narrow, lens)
    table = torch.full((batch, 2500), -1, dtype=torch.int32)
    table[:, :narrow.shape[1]] = narrow
    q = pool.randn((batch, 24, dim), 2.0)
    got = attend(device, pool, table, lens, q, dim ** -0.5)
    R.check(got, *R.attention(pool, narrow, lens, q, dim ** -0.5))


def test_attention_of_many_sequences(device):
    """More sequences than a wave has lanes, lengths of every order, one far longer than the others."""
    g = torch.Generator().manual_seed(9)
    lens = [int(2.0 ** (10 * float(torch.rand((), generator=g)))) - 1 for _ in range(150)]
    lens[70], lens[3], lens[149] = 9000, 0, 0
    pool = R.Pool("fp16", sum(-(-n // 16) for n in lens) + 1, 1, 16, 64, seed=10, bounds=False)
    table = pool.tables(lens)
    poison(pool, table, lens)
    q = pool.randn((150, 2, 64), 2.0)
    got = attend(device, pool, table, lens, q, 0.125)
    R.check(got, *R.attention(pool, table, lens, q, 0.125))


@pytest.mark.parametrize("scale", [0.125, -0.25, 0.0, 3.0])
def test_scales_and_peaked_scores(device, scale):
    """Scores of hundreds, one far over the others late in the window, and scales of either sign."""
    for kind in ("fp16", "int8"):
        pool = R.Pool(kind, 60, 2, 16, 64, seed=12, bounds=False)
        table = pool.tables([900])
        if kind == "fp16":
            pool.k[int(table[0, 50]), :, 3] *= 12
        q = pool.randn((1, 8, 64), 6.0)
        got = attend(device, pool, table, [900], q, scale)
        R.check(got, *R.attention(pool, table, [900], q, scale), kind)


def test_values_of_very_different_rows(device):
    """8-bit rows whose scales lie 2^30 apart: no weight is lost or overflows."""
    for kind in ("int8", "e4m3"):
        pool = R.Pool(kind, 60, 2, 16, 64, seed=13, bounds=False)
        table = pool.tables([700])
        pool.v_scale *= 2.0 ** torch.randint(-24, 6, pool.v_scale.shape, generator=pool.g).float()
        q = pool.randn((1, 8, 64))
        got = attend(device, pool, table, [700], q, 0.125)
        R.check(got, *R.attention(pool, table, [700], q, 0.125), kind)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("where", ["v_inf", "v_both", "v_nan", "k_inf", "k_minus", "k_nan", "all_minus", "v_inf_far", "v_inf_near"])
def test_infinities_and_nan(device, dim, where):
    """What a 64-bit softmax gives: infinite values stay infinite, a NaN score makes its heads NaN, others are untouched."""
    lens = [100, 700, 1500]
    pool = R.Pool("fp16", 200, 2, 16, dim, seed=20, bounds=False)
    table = pool.tables(lens)
    poison(pool, table, lens)
    pool.k.abs_()
    q = pool.randn((3, 8, dim)).abs()
    q[:, ::2] *= -1
    at = lambda t: (int(table[1, t // 16]), 1, t % 16)
    if where == "v_inf":
        pool.v[at(5)][3] = math.inf
    elif where == "v_both":
        pool.v[at(5)][3], pool.v[at(650)][3], pool.v[at(650)][4] = math.inf, -math.inf, -math.inf
    elif where == "v_nan":
        pool.v[at(699)][3] = math.nan
    elif where == "k_inf":
        pool.k[at(300)][7] = math.inf
    elif where == "k_minus":
        pool.k[at(300)][7] = -math.inf
    elif where == "k_nan":
        pool.k[at(0)][7] = math.nan
    elif where == "all_minus":
        for t in range(700):
            pool.k[at(t)][0] = -math.inf
    elif where == "v_inf_near":
        # scores about 0.57 sqrt(D) k: 46 apart, a weight of 1e-20, below fp16's range but not fp32's
        pool.k[at(9)] = 0.01
        q[1] = 0.5 + q[1].abs() * 0.1
        pool.k[at(10)] = 80 / dim ** 0.5
        pool.v[at(9)][3] = math.inf
    elif where == "v_inf_far":
        # 185 apart: a weight below fp32's range
        pool.k[at(9)] = 0.01
        q[1] = 0.5 + q[1].abs() * 0.1
        pool.k[at(10)] = 40.0 * 8 / dim ** 0.5
        pool.v[at(9)][3] = math.inf
    got = attend(device, pool, table, lens, q, dim ** -0.5)
    R.check(got, *R.attention(pool, table, lens, q, dim ** -0.5), where)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_every_code(device, kind):
    """All 256 codes as K and V: int8 from -128, e4m3 with its subnormal numbers; a NaN code makes its heads NaN."""
    pool = R.Pool(kind, 40, 2, 16, 64, seed=21, bounds=False)
    lens = [600]
    table = pool.tables(lens)
    codes = torch.arange(40 * 2 * 16 * 64).view(40, 2, 16, 64) * 37 % 256
    if kind == "e4m3":
        codes = torch.where(codes % 128 == 127, codes - 1, codes)
    pool.k.view(torch.uint8).copy_(codes)
    pool.v.view(torch.uint8).copy_(codes.flip(3))
    q = pool.randn((1, 8, 64), 0.3)
    R.check(attend(device, pool, table, lens, q, 0.125), *R.attention(pool, table, lens, q, 0.125))
    if kind == "e4m3":
        for name, at in (("k", 70), ("v", 599)):
            kept = getattr(pool, name).clone()
            getattr(pool, name).view(torch.uint8)[int(table[0, at // 16]), 1, at % 16, 5] = 0xff
            got = attend(device, pool, table, lens, q, 0.125)
            R.check(got, *R.attention(pool, table, lens, q, 0.125), name)
            assert torch.isnan(got[0, 4:]).any() and not torch.isnan(got[0, :4]).any()
            setattr(pool, name, kept)


@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("batch, heads, tokens, count, size", [(1, 200, 10007, 0, 16), (8, 128, 9000, 80, 64),
                                                               (2, 100, 20000, 0, 128)])
def test_chunks_of_many_tiles(device, kind, batch, heads, tokens, count, size):
    """So many heads that a wave takes more tiles than it looks pages up for at once (against 64 bits on the device)."""
    K = kernels()
    dim = 64
    pool = R.Pool(kind, 30, heads, size, dim, seed=heads, bounds=False)
    width = -(-tokens // size)
    table = torch.randint(0, 30, (batch, width), generator=pool.g, dtype=torch.int32)
    q = pool.randn((batch, heads * 2, dim), 2.0).to(device)
    lens = [tokens - 7 * b for b in range(batch)]
    chosen = None
    if count:
        chosen = torch.stack([torch.randperm(width, generator=pool.g)[:count].sort().values
                              for _ in range(batch * heads)]).view(batch, heads, count).int()
    got = K.paged_attention(q, pool.pages(device), table.to(device), i32(lens, device), 0.125,
                            None if chosen is None else chosen.to(device)).double()
    kk, vv = pool.values("k").to(device), pool.values("v").to(device)
    for b in range(batch):
        for h in range(0, heads, 7):
            ords = torch.arange(width) if chosen is None else chosen[b, h].long()
            pos = (ords[:, None] * size + torch.arange(size)).reshape(-1).to(device) < lens[b]
            page = table[b].long()[ords].to(device)
            k, v = (x[page, h].reshape(-1, dim)[pos] for x in (kk, vv))
            for g in range(2):
                x = q[b, 2 * h + g].double()
                want = torch.softmax((k * x).sum(-1) * 0.125, 0) @ v
                size_qk = float(((k * x).abs().sum(-1) * 0.125).max())
                tol = want.abs() * 2.0 ** -11 + 2.0 ** -25 + float(v.abs().max()) * (
                    2 * 68 * 2.0 ** -24 * size_qk + 2 * len(k) * 2.0 ** -24 + 2.0 ** -16)  # as in R.attention
                assert ((got[b, 2 * h + g] - want).abs() <= tol).all(), (b, h, g)


def test_small_weights_of_a_very_long_sequence(device):
    """One position with a value of 0 and 2^24 - 1 with 2^-33.5 of its weight and a value of 2^15, in fp16 pages, and so
    many heads that the chip is full without cutting the sequence.  The wave that sees the first position loses the
    others' weights, which are below fp16's range there; every other wave goes by its own largest weight.

    The tolerance: the wave with the first position drops up to 2^20 weights of up to 2^-33; fp16's half step of the
    output; 2^-16 of it for the weights' exponent (a score of 33.5 in base 2 is off by 2^-18) and roundings."""
    K = kernels()
    heads, tokens, dim = 512, 1 << 24, 64
    k, v = (torch.zeros((2, heads, 16, dim), dtype=D16, device=device) for _ in range(2))
    v[:] = 32768.0
    v[0, :, 0] = 0.0
    k[0, :, 0, 0] = 23.21875
    table = torch.ones((1, tokens // 16), dtype=torch.int32, device=device)
    table[0, 0] = 0
    q = torch.zeros((1, heads, dim), dtype=D16, device=device)
    q[:, :, 0] = 1.0
    got = K.paged_attention(q, K.KVPages(k, v), table, i32([tokens], device), 1.0).double()
    w = math.exp(-23.21875)
    want = 32768.0 * (tokens - 1) * w / (1.0 + (tokens - 1) * w)
    off = float((got - want).abs().max())
    assert off <= 2.0 ** 20 * 2.0 ** -33 * 32768 + want * (2.0 ** -11 + 2.0 ** -16), (off, want)


# ------------------------------------------------------------------ page choice

@pytest.mark.parametrize("dim, heads, group, size, count, first, last", [
    (64, 8, 4, 16, 4, 1, 1), (64, 2, 1, 16, 300, 1, 1), (128, 3, 8, 32, 7, 0, 0), (256, 1, 3, 16, 20, 3, 2),
    (64, 1, 20, 64, 3, 0, 3), (128, 2, 4, 16, 33, 0, 1)])
def test_select_and_attend(device, dim, heads, group, size, count, first, last):
    lens = [0, 1, size, size + 1, 1900, 2500, 333]
    pool = R.Pool("int8", sum(-(-n // size) for n in lens) + 2, heads, size, dim, seed=count)
    table = pool.tables(lens)
    poison(pool, table, lens)
    q = pool.randn((len(lens), heads * group, dim))
    K = kernels()
    chosen = K.page_select(q.to(device), pool.pages(device), table.to(device), i32(lens, device), count, first=first,
                           last=last)
    want = R.select(pool, table, lens, q, count, first, last)
    assert torch.equal(chosen.cpu(), want)
    got = attend(device, pool, table, lens, q, dim ** -0.5, chosen)
    R.check(got, *R.attention(pool, table, lens, q, dim ** -0.5, want))


def test_select_ties_infinities_and_missing_pages(device):
    """Equal scores go to the lower page, NaN counts as infinite, a table entry that is no page is the last choice."""
    K = kernels()
    pool = R.Pool("fp16", 80, 2, 16, 64, seed=31)
    lens = [1200, 640]
    pool.bounds[:] = torch.tensor([-1.0, 1.0]).half()[None, None, :, None]
    table = torch.arange(80, dtype=torch.int32).view(1, 80).repeat(2, 1)
    table[1, 5], table[1, 6] = -1, 80
    q = pool.randn((2, 4, 64))
    for edit in range(5):
        if edit == 1:
            pool.bounds[40, :, 1, 2] = math.nan
            pool.bounds[40, :, 0, 2] = math.nan
        elif edit == 2:
            pool.bounds[50, 0, 1, 9] = math.inf
        elif edit == 3:
            pool.bounds[20, :, 0] = -math.inf
            pool.bounds[20, :, 1] = -math.inf
        elif edit == 4:
            q[0, 0, 0] = math.nan
        for count, first, last in ((1, 0, 0), (2, 1, 1), (9, 2, 3), (39, 0, 1), (40, 0, 0), (75, 1, 1), (90, 1, 1)):
            got = K.page_select(q.to(device), pool.pages(device), table.to(device), i32(lens, device), count,
                                first=first, last=last)
            assert torch.equal(got.cpu(), R.select(pool, table, lens, q, count, first, last)), (edit, count)


def test_long_rows_of_pages(device):
    """A sequence of many thousand pages: the choice over more pages than a block has threads."""
    K = kernels()
    pages, n = 40, 20000
    pool = R.Pool("fp16", pages, 1, 16, 64, seed=33)
    table = torch.randint(0, pages, (1, n), generator=pool.g, dtype=torch.int32)
    q = pool.randn((1, 2, 64))
    lens = [n * 16 - 5]
    score = R.select(pool, torch.arange(pages, dtype=torch.int32)[None], [pages * 16], q, pages, 0, 0)
    assert score.shape[-1] == pages
    for count in (5, 2500):
        got = K.page_select(q.to(device), pool.pages(device), table.to(device), i32(lens, device), count)
        assert torch.equal(got.cpu(), R.select(pool, table, lens, q, count, 1, 1))


def test_lists_of_the_callers_own(device):
    """Lists with pages twice, past the sequence, negative, and in any order: each listed page counts as often as it is listed."""
    pool = R.Pool("fp16", 90, 2, 16, 64, seed=34)
    lens = [1000, 39, 0]
    table = pool.tables(lens)
    poison(pool, table, lens)
    table[0, 7] = 4000  # no page
    q = pool.randn((3, 4, 64))
    chosen = torch.randint(-3, 70, (3, 2, 50), generator=pool.g, dtype=torch.int32)
    chosen[1, 0] = torch.tensor([2, 2, 2147483647, -2147483648] + [-1] * 46, dtype=torch.int32)
    got = attend(device, pool, table, lens, q, 0.125, chosen)
    R.check(got, *R.attention(pool, table, lens, q, 0.125, chosen))
    assert not attend(device, pool, table, lens, q, 0.125, chosen[:, :, :0]).any()


# ------------------------------------------------------------------ layouts, streams, graphs

def test_strided_pools_and_tables(device):
    """K and V as slices of one pool of several layers, a table that is a slice of a wider one."""
    K = kernels()
    lens = [700, 33]
    pool = R.Pool("fp16", 50, 3, 16, 64, seed=41)
    table = pool.tables(lens)
    q = pool.randn((2, 6, 64))
    joint = torch.full((50, 2, 2, 3, 16, 64), math.nan, dtype=D16, device=device)  # pages, layers, K/V, ...
    joint[:, 1, 0], joint[:, 1, 1] = pool.k.to(device), pool.v.to(device)
    heads_first = torch.full((2, 3, 50, 16, 64), math.nan, dtype=D16, device=device)
    heads_first[0], heads_first[1] = pool.k.transpose(0, 1).to(device), pool.v.transpose(0, 1).to(device)
    wide = torch.full((2, 200), 7, dtype=torch.int32, device=device)
    wide[:, 20:20 + table.shape[1]] = table.to(device)
    want = R.attention(pool, table, lens, q, 0.125)
    for k, v in ((joint[:, 1, 0], joint[:, 1, 1]), (heads_first[0].transpose(0, 1), heads_first[1].transpose(0, 1))):
        pages = K.KVPages(k, v, bounds=pool.bounds.to(device))
        got = K.paged_attention(q.to(device), pages, wide[:, 20:20 + table.shape[1]], i32(lens, device), 0.125)
        R.check(got, *want)
        row = pool.randn((2, 3, 64)).to(device)
        K.paged_append(pages, wide[:, 20:20 + table.shape[1]], i32([0, 32], device), row, row)
        assert torch.equal(k[int(table[0, 0]), :, 0], row[0]) and torch.equal(v[int(table[1, 2]), :, 0], row[1])
    assert torch.isnan(joint[:, 0]).all()
    # queries that are a slice, on an address that is not 16-byte aligned
    flat = torch.zeros(2 * 6 * 64 + 1, dtype=D16, device=device)
    flat[1:] = q.to(device).reshape(-1)
    pages = K.KVPages(joint[:, 1, 0], joint[:, 1, 1])
    a = K.paged_attention(flat[1:].view(2, 6, 64), pages, table.to(device), i32(lens, device), 0.125)
    b = K.paged_attention(q.to(device), pages, table.to(device), i32(lens, device), 0.125)
    assert torch.equal(a, b)


def test_results_do_not_depend_on_the_table_s_width_or_the_batch(device):
    """A wider table, and a batch that holds other sequences as well, change a result by rounding alone."""
    K = kernels()
    lens = [2000, 17]
    pool = R.Pool("fp16", 140, 2, 16, 64, seed=43, bounds=False)
    table = pool.tables(lens)
    q = pool.randn((2, 8, 64))
    want = R.attention(pool, table, lens, q, 0.125)
    pages = pool.pages(device)
    for width in (table.shape[1], 4096):
        t = torch.full((2, width), -1, dtype=torch.int32)
        t[:, :table.shape[1]] = table
        first = K.paged_attention(q.to(device), pages, t.to(device), i32(lens, device), 0.125)
        R.check(first, *want, str(width))
        for _ in range(3):  # and repeats bit for bit
            assert torch.equal(first, K.paged_attention(q.to(device), pages, t.to(device), i32(lens, device), 0.125))


def test_long_pools_pass_32_bit_offsets(device):
    """Rows past 2^32 elements into the pool are written, read and attended."""
    K = kernels()
    heads, size, dim = 8, 128, 256
    pages = (1 << 32) // (heads * size * dim) + 40
    if torch.cuda.mem_get_info()[0] < 5 * pages * heads * size * dim * 2:
        pytest.skip("needs 40 GB")
    k = torch.empty((pages, heads, size, dim), dtype=D16, device=device)
    v = torch.empty_like(k)
    pool = K.KVPages(k, v, bounds=torch.zeros((pages, heads, 2, dim), dtype=D16, device=device))
    g = torch.Generator().manual_seed(3)
    rows = [torch.randn((300, heads, dim), generator=g).half() for _ in range(2)]
    table = i32([[pages - 1, 2, pages - 30]], device)
    cu = i32([0, 300], device)
    K.paged_append(pool, table, i32([0], device), rows[0].to(device), rows[1].to(device), cu)
    ko, vo = K.paged_read(pool, table, i32([0], device), cu, 300)
    assert torch.equal(ko.cpu(), rows[0]) and torch.equal(vo.cpu(), rows[1])
    q = torch.randn((1, heads, dim), generator=g).half()
    small = R.Pool("fp16", 3, heads, size, dim, seed=1, bounds=False)
    at = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    small.append(at, [0], *rows, [0, 300])
    R.check(K.paged_attention(q.to(device), pool, table, i32([300], device), 0.0625),
            *R.attention(small, at, [300], q, 0.0625))
    chosen = K.page_select(q.to(device), pool, table, i32([300], device), 2)
    assert chosen[0, :, 0].eq(0).all() and chosen[0, :, 1].eq(2).all()


@pytest.mark.parametrize("kind", ["fp16", "int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens, times", [([2100, 0, 33, 700], 1), ([16, 0, 77, 5], 300)])
def test_pools_past_the_last_level_cache(device, kind, dim, lens, times):
    """300 MB of pages with the sequences' scattered over them, and room for all of them in the table: their rows
    are loaded as used once, in chunks by the lengths and in one for each of many sequences, which share pages."""
    K = kernels()
    heads, size = 4, 16
    pool = R.Pool(kind, sum(-(-n // size) for n in lens) + 1, heads, size, dim, seed=dim + len(lens), bounds=False)
    near = pool.tables(lens)
    poison(pool, near, lens)
    q = pool.randn((len(lens), 12, dim), 2.0)
    count = 300_000_000 // (2 * heads * size * dim * pool.k.element_size())
    to = torch.randperm(count, generator=pool.g)[:pool.count].int()
    small = pool.pages(device)
    far = [None if x is None else x.new_zeros((count, *x.shape[1:])) for x in small]
    for big, x in zip(far, small):
        if x is not None:
            big.view(torch.uint8)[to.to(device).long()] = x.view(torch.uint8)
    table = torch.full((len(lens), max(near.shape[1], -(-count // (len(lens) * times)))), -1, dtype=torch.int32)
    table[:, :near.shape[1]] = torch.where(near >= 0, to[near.clamp(min=0).long()], near)
    got = K.paged_attention(q.repeat(times, 1, 1).to(device), K.KVPages(*far), table.repeat(times, 1).to(device),
                            i32(lens * times, device), dim ** -0.5)
    R.check(got, *(x.repeat(times, 1, 1) for x in R.attention(pool, near, lens, q, dim ** -0.5)))


@pytest.mark.parametrize("kind", ["fp16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 256])
def test_what_the_caller_says_is_held_changes_no_bit(device, kind, dim):
    """A pool of 300 MB with a few of its pages in use: the number of those, a far larger one or none; and many queries
    over one sequence's pages, whose table is a row of stride 0."""
    K = kernels()
    count = 300_000_000 // (2 * 4 * 64 * dim * (2 if kind == "fp16" else 1))
    small = R.Pool(kind, 60, 4, 64, dim, seed=dim, bounds=False)
    lens = [3000, 0, 17, 555]
    near = small.tables(lens)
    poison(small, near, lens)
    q = small.randn((4, 16, dim), 2.0)
    far = [None if x is None else torch.cat([x.new_zeros((count - 60, *x.shape[1:])), x]) for x in
           (None if x is None else x.view(torch.uint8) if x.element_size() == 1 else x for x in small.pages(device))]
    pages = K.KVPages(*(x if y is None or y.element_size() > 1 else x.view(y.dtype) for x, y in zip(far, small.pages(device))))
    table = torch.full((4, count // 4 + 1), -1, dtype=torch.int32)
    table[:, :near.shape[1]] = torch.where(near >= 0, near + count - 60, near)
    table, n = table.to(device), i32(lens, device)
    got = [K.paged_attention(q.to(device), pages, table, n, dim ** -0.5, None, held) for held in (0, 60, 1 << 30)]
    R.check(got[0], *R.attention(small, near, lens, q, dim ** -0.5))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    ends = [1 + 97 * i for i in range(30)]
    q = small.randn((30, 16, dim), 2.0)
    got = K.paged_attention(q.to(device), pages, table[:1].expand(30, -1), i32(ends, device), dim ** -0.5)
    R.check(got, *R.attention(small, near[:1].expand(30, -1), ends, q, dim ** -0.5))
    for held in (-1, 1 << 31):
        with pytest.raises(ValueError, match="held_pages"):
            K.paged_attention(q.to(device), pages, table[:1].expand(30, -1), i32(ends, device), 0.1, None, held)


def test_another_stream(device):
    K = kernels()
    pool = R.Pool("int8", 120, 2, 16, 64, seed=45)
    lens = [1700]
    table = pool.tables(lens)
    q = pool.randn((1, 8, 64))
    pages, t, n, qd = pool.pages(device), table.to(device), i32(lens, device), q.to(device)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        chosen = K.page_select(qd, pages, t, n, 10)
        got = K.paged_attention(qd, pages, t, n, 0.125, chosen)
    s.synchronize()
    R.check(got, *R.attention(pool, table, lens, q, 0.125, R.select(pool, table, lens, q, 10, 1, 1)))


def test_captured_step(device):
    """A decode step in a graph: replays follow the lengths and rows that the program writes, among eager calls."""
    K = kernels()
    B, H, size = 3, 2, 16
    start = [5, 0, 1500]
    pool = R.Pool("int8", 140, H, size, 64, seed=50)
    table = pool.tables([n + 40 for n in start])
    pages, t, lens = pool.pages(device), table.to(device), i32(start, device)
    k, v, q = (torch.zeros((B, n, 64), dtype=D16, device=device) for n in (H, H, 8))

    def step():
        K.paged_append(pages, t, lens, k, v)
        lens.add_(1)
        return (K.paged_attention(q, pages, t, lens, 0.125),
                K.paged_attention(q, pages, t, lens, 0.125, K.page_select(q, pages, t, lens, 6)))

    keep = [x.clone() for x in pages] + [lens.clone()]
    step()
    for x, y in zip(list(pages) + [lens], keep):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dense, sparse = step()
    for x, y in zip(list(pages) + [lens], keep):
        x.copy_(y)
    now = list(start)
    for i in range(20):
        rows = [pool.randn((B, n, 64)) for n in (H, H, 8)]
        for x, r in zip((k, v, q), rows):
            x.copy_(r)
        graph.replay()
        pool.append(table, now, rows[0], rows[1], [0, 1, 2, 3])
        now = [n + 1 for n in now]
        if i % 5 == 0 or i > 16:
            R.check(dense, *R.attention(pool, table, now, rows[2], 0.125), f"replay {i}")
            R.check(sparse, *R.attention(pool, table, now, rows[2], 0.125, R.select(pool, table, now, rows[2], 6, 1, 1)))
            torch.zeros(1 << 20, device=device).sum().item()  # the program's own work between replays
            assert torch.equal(dense, K.paged_attention(q, pages, t, lens, 0.125))
    assert lens.tolist() == now


def test_wrappers_refuse(device):
    K = kernels()
    pool = R.Pool("fp16", 8, 2, 16, 64, seed=60)
    pages, t, n = pool.pages(device), torch.zeros((2, 4), dtype=torch.int32, device=device), i32([5, 6], device)
    q = torch.zeros((2, 4, 64), dtype=D16, device=device)
    rows = q[:, :2].contiguous()
    cu = i32([0, 1, 2], device)
    s = torch.zeros((8, 2, 16), device=device)
    half = K.KVPages(pages.k, pages.v)
    bad = [
        lambda: K.paged_attention(q.float(), pages, t, n, 0.1), lambda: K.paged_attention(q[:1], pages, t, n, 0.1),
        lambda: K.paged_attention(q[:, :3], pages, t, n, 0.1), lambda: K.paged_attention(q[:, :, :32], pages, t, n, 0.1),
        lambda: K.paged_attention(q, pages, t.long(), n, 0.1), lambda: K.paged_attention(q, pages, t, n.long(), 0.1),
        lambda: K.paged_attention(q, pages, t, n[:1], 0.1), lambda: K.paged_attention(q, pages, t[:1], n, 0.1),
        lambda: K.paged_attention(q, pages, t.t().contiguous().t(), n, 0.1),
        lambda: K.paged_attention(q, pages, t, n, math.inf), lambda: K.paged_attention(q, pages, t, n, 3e38),
        lambda: K.paged_attention(q, pages._replace(k_scale=s), t, n, 0.1),
        lambda: K.paged_attention(q, pages._replace(v=pages.v.to(torch.int8)), t, n, 0.1),
        lambda: K.paged_attention(q, pages._replace(k=pages.k.bfloat16(), v=pages.v.bfloat16()), t, n, 0.1),
        lambda: K.paged_attention(q, pages._replace(k=pages.k.to(torch.int8), v=pages.v.to(torch.int8)), t, n, 0.1),
        lambda: K.paged_attention(q, pages._replace(k=pages.k[..., ::2], v=pages.v[..., ::2]), t, n, 0.1),
        lambda: K.paged_attention(q, pages._replace(k=pages.k[:, :, :8], v=pages.v[:, :, :8]), t, n, 0.1),
        lambda: K.paged_attention(q, pages, t.cpu(), n, 0.1), lambda: K.paged_attention(q.cpu(), pages, t, n, 0.1),
        lambda: K.paged_attention(q, pages, t, n, 0.1, torch.zeros((2, 4, 3), dtype=torch.int32, device=device)),
        lambda: K.paged_attention(q, pages, t, n, 0.1, torch.zeros((2, 2, 3), device=device)),
        lambda: K.page_select(q, half, t, n, 3), lambda: K.page_select(q, pages, t, n, 1),
        lambda: K.page_select(q, pages, t, n, 0, first=0, last=0), lambda: K.page_select(q, pages, t, n, 3, first=-1),
        lambda: K.page_select(q, pages._replace(bounds=pages.bounds.float()), t, n, 3),
        lambda: K.paged_append(pages, t, n, rows[:1], rows[:1]), lambda: K.paged_append(pages, t, n, rows, rows[:, :1]),
        lambda: K.paged_append(pages, t, n, rows.float(), rows.float()),
        lambda: K.paged_append(pages, t, n, rows, rows, cu[:2]), lambda: K.paged_append(pages, t, n, rows, rows, cu.long()),
        lambda: K.paged_read(pages, t, n, cu, -1), lambda: K.paged_read(pages, t, n, cu.cpu(), 2),
        lambda: K.paged_read(pages, t, n, cu, 2, (rows, rows.float()))]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was accepted")


# ------------------------------------------------------------------ the cache

@pytest.mark.parametrize("kind, dim, size", [("fp16", 64, 16), ("int8", 128, 32), ("e4m3", 64, 64), ("fp16", 256, 16)])
def test_cache_serves_a_batch(device, kind, dim, size):
    """Prompts in chunks, decode steps, a sequence that ends and one that takes its place: every output against
    attention over the rows as they are held, and no page of another's is touched."""
    from apple_amd.paged import RFSNPagedKVCache
    from apple_amd.storage import RFSNConfig

    cfg = RFSNConfig(hidden_dim=8 * dim, num_heads=8, num_kv_heads=2, head_dim=dim, num_subspaces=8, subspace_dim=dim // 8)
    cache = RFSNPagedKVCache(cfg, batch=3, pages=1500 // size, page_size=size, page_type=kind, device=device)
    g = torch.Generator().manual_seed(dim)
    rand = lambda *s: torch.randn(s, generator=g).half()
    model = R.Pool(kind, 1500 // size, 2, size, dim, seed=1)
    held = [0, 0, 0]

    def mirror():
        """The pool as it lies on the device, in the restatement."""
        for name, t in cache.pages._asdict().items():
            if t is not None:
                setattr(model, name, t.cpu())
        assert cache.num_tokens == held == cache.lens.tolist()
        return cache.table.cpu()

    def append(rows, counts):
        k, v = rand(rows, 2, dim), rand(rows, 2, dim)
        t0 = [list(r) for r in cache._held]
        before = mirror()
        assert before is not None and t0 is not None
        cache.append(k.to(device), v.to(device), counts)
        each = counts if counts is not None else [1, 1, 1]
        cu = [0]
        for c in each:
            cu.append(cu[-1] + c)
        model.append(cache.table.cpu(), held, k, v, cu)
        for b, c in enumerate(each):
            held[b] += c
        for name, t in cache.pages._asdict().items():
            if t is not None:
                assert same(t, getattr(model, name)), name

    append(130, [100, 0, 30])
    append(520, [0, 517, 3])
    q = rand(5, 8, dim)
    out = cache.prompt_attention(1, q.to(device))
    window = [x.cpu() for x in cache.sequence_window(1)]
    wk, wv, _ = model.window(cache.table.cpu(), 1, 0, 517)
    for got, want in zip(window, (wk, wv)):
        assert ((got.double() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -24) + 2.0 ** -25).all()
    one = R.Pool("fp16", -(-517 // size), 2, size, dim, seed=2, bounds=False)
    at = torch.arange(one.count, dtype=torch.int32)[None]
    one.append(at, [0], window[0], window[1], [0, 517])
    for i in range(5):
        want, tol = R.attention(one, at, [513 + i], q[i:i + 1], dim ** -0.5)
        R.check(out[i:i + 1], want, tol + 2.0 ** -11 * want.abs().amax())  # its own kernel's fp16 weights and steps
    for i in range(size + 2):
        append(3, None)
        if i % 7 == 0 or i == size + 1:
            q = rand(3, 8, dim)
            t = mirror()
            R.check(cache.attention_forward(q.to(device)), *R.attention(model, t, held, q, dim ** -0.5))
            want = R.select(model, t, held, q, 4, 1, 1)
            R.check(cache.attention_forward(q.to(device), sparse_pages=4), *R.attention(model, t, held, q, dim ** -0.5, want))
    free = cache.free_pages
    cache.release(1)
    held[1] = 0
    assert cache.free_pages > free
    q = rand(3, 8, dim)
    got = cache.attention_forward(q.float().to(device))
    assert got.dtype == torch.float32 and not got[1].any()
    R.check(got[[0, 2]].half(), *(x[[0, 2]] for x in R.attention(model, mirror(), held, q, dim ** -0.5)))
    append(40, [0, 40, 0])
    q = rand(3, 8, dim)
    R.check(cache.attention_forward(q.to(device)), *R.attention(model, mirror(), held, q, dim ** -0.5))
