"""What bounds a paged cache's memory, on the GPU against the restatement in 64
bits: 4-bit pages, accumulated attention weights, eviction, rotary positions, and
all of them together as a cache runs them."""

import math

import pytest
import torch

from tests import bounded_reference as B
from tests import paged_reference as R
from tests.test_gpu_paged import D16, i32, kernels, same

pytestmark = pytest.mark.gpu

CU = lambda counts: [sum(counts[:i]) for i in range(len(counts) + 1)]


def alike(pool, pages, weight=None):
    for name, got in pages._asdict().items():
        if got is not None:
            assert same(got, getattr(pool, name)), name
    if weight is not None:
        assert same(weight, pool.weight), "weight"


# ------------------------------------------------------------------ 4-bit rows

@pytest.mark.parametrize("dim, heads, size, starts, counts, pad", [
    (64, 8, 16, [0], [1], 0), (64, 2, 16, [15, 16, 0, 31], [1, 1, 1, 1], 0), (64, 5, 32, [3, 0, 40], [70, 0, 9], 5),
    (128, 3, 64, [0, 63, 64], [64, 2, 200], 3), (256, 1, 16, [7, 0], [33, 1], 0), (256, 6, 256, [250], [300], 1),
    (128, 4, 128, [0, 0, 0, 100], [0, 0, 0, 29], 9), (64, 1, 16, [0], [1000], 0), (64, 40, 16, [3], [700], 2)])
def test_append_and_read(device, dim, heads, size, starts, counts, pad):
    K = kernels()
    ends = [a + n for a, n in zip(starts, counts)]
    pool = B.Pool("e2m1", sum(-(-e // size) for e in ends) + 2, heads, size, dim, seed=dim + size)
    table, n = pool.tables(ends), sum(counts)
    k, v = pool.randn((n + pad, heads, dim), 3.0), pool.randn((n + pad, heads, dim))
    k[0, 0] = 0
    pages, weight = pool.pages(device), pool.weight.to(device)
    one = all(c == 1 for c in counts) and not pad
    wide = torch.zeros((n + pad, 2, heads, dim), dtype=D16, device=device)  # parts of a projection's output
    wide[:, 0], wide[:, 1] = k.to(device), v.to(device)
    K.paged_append(pages, table.to(device), i32(starts, device), wide[:, 0], wide[:, 1], None if one else i32(CU(counts), device),
                   weight=weight)
    pool.append(table, starts, k, v, CU(counts))
    alike(pool, pages, weight)
    for begin in (starts, [0] * len(starts)):
        at = CU([e - a for a, e in zip(begin, ends)])
        ko, vo = K.paged_read(pages, table.to(device), i32(begin, device), i32(at, device), at[-1] + 2)
        for b in range(len(starts)):
            wk, wv, _ = pool.window(table, b, begin[b], ends[b])
            for got, want in ((ko, wk), (vo, wv)):  # exact in fp16
                assert torch.equal(got[at[b]:at[b + 1]].cpu().double(), want)
        assert not ko[at[-1]:].any() and not vo[at[-1]:].any()


def test_every_code_and_scale_read_back(device):
    """256 bytes of codes under 256 scales: code * scale, NaN under those that are none (infinite under 248)."""
    K = kernels()
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)                # [scale, codes]: 512 coordinates
    k = codes.view(256, 1, 4, 2, 32).permute(0, 1, 3, 2, 4).reshape(128, 1, 16, 32).contiguous()
    scale = torch.arange(256, dtype=torch.uint8).repeat_interleave(8).view(128, 1, 16, 1).expand(-1, -1, -1, 4).contiguous()
    pages = K.KVPages(*(t.to(device) for t in (k, k, scale, scale)))
    table, at = torch.arange(128, dtype=torch.int32, device=device)[None], i32([0, 2048], device)
    ko, vo = K.paged_read(pages, table, at[:1], at, 2048)
    want = B.values4(k, scale)[:, 0].reshape(2048, 64)
    assert same(ko[:, 0], want.half()) and same(vo[:, 0], want.half())


def test_midpoints_and_borders_of_the_codes(device):
    """Every midpoint of two codes under every mantissa of a scale, the fp16 neighbours of each, and the scale's own midpoints."""
    K = kernels()
    rows = []
    for e in (-17, -14, -9, 0, 7, 13):
        for m in range(8, 16):
            scale = m * 2.0 ** (e - 3) if e >= -14 else m * 2.0 ** -17
            if 6 * scale > 65504:
                continue
            mids = [scale * x for x in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)]
            for top in (6 * scale, 6 * scale * (1 + 1 / 64), 6 * scale * (1 - 1 / 64)):
                base = torch.tensor([top] + mids + [-x for x in mids] + [0.0], dtype=torch.float64).half()
                bits = base.view(torch.int16)
                for step in (0, 1, -1):
                    near = bits + torch.where((bits & 0x7FFF) > 0, step, 0).to(torch.int16)
                    near[0] = bits[0]
                    rows.append(near.view(D16))
    for amax in range(1, 300):  # the smallest groups, where scales are multiples of 2^-17 or none
        rows.append(torch.linspace(-1, 1, 16, dtype=torch.float64).mul(amax * 2.0 ** -24).half())
    for x in (65504.0, 61440.0, 63000.0, 62976.0, 30000.0, 2.0 ** -14 * 6, 6.1e-5, -0.0):
        rows.append(torch.linspace(x, -x / 2, 16, dtype=torch.float64).half())
    rows += [torch.zeros(16, dtype=D16)] * (-len(rows) % 4)
    x = torch.stack(rows).reshape(-1, 1, 64)
    n = len(x)
    pool = B.Pool("e2m1", -(-n // 16), 1, 16, 64, seed=1, bounds=False)
    table = torch.arange(pool.count, dtype=torch.int32)[None]
    pages = pool.pages(device)
    K.paged_append(pages, table.to(device), i32([0], device), x.to(device), (-x).to(device), i32([0, n], device))
    pool.append(table, [0], x, -x, [0, n])
    alike(pool, pages)


def test_groups_that_are_not_finite(device):
    """Scale NaN for 16 coordinates, the row's others as they are."""
    K = kernels()
    pool = B.Pool("e2m1", 3, 2, 16, 128, seed=5)
    k, v = pool.randn((6, 2, 128)), pool.randn((6, 2, 128))
    k[1, 0, 3], k[2, 1, 127], v[3, 0, 16], v[4, 1, 15] = math.inf, math.nan, -math.inf, math.nan
    table = torch.tensor([[1, 2]], dtype=torch.int32)
    pages = pool.pages(device)
    K.paged_append(pages, table.to(device), i32([12], device), k.to(device), v.to(device), i32([0, 6], device))
    pool.append(table, [12], k, v, [0, 6])
    alike(pool, pages)
    ko, vo = K.paged_read(pages, table.to(device), i32([12], device), i32([0, 6], device), 6)
    assert torch.isnan(ko[1, 0, :16]).all() and torch.isfinite(ko[1, 0, 16:]).all() and torch.isnan(ko[2, 1, 112:]).all()
    assert torch.isnan(vo[3, 0, 16:32]).all() and int(torch.isnan(vo).sum()) == 32


@pytest.mark.parametrize("batch", [5, 70])
def test_any_row_offsets_stay_in_the_tables_pages(device, batch):
    """Lengths, offsets and entries that are no such thing write nothing outside the pages that the table names."""
    K = kernels()
    pool = B.Pool("e2m1", 300, 3, 16, 64, seed=batch)
    g = torch.Generator().manual_seed(batch)
    table = torch.full((batch, 3), -1, dtype=torch.int32)
    table[:, :2] = torch.randperm(280, generator=g)[:2 * batch].view(batch, 2).int()
    table[1] = torch.tensor([99999, -5, 2147483647])
    pages, weight = pool.pages(device), pool.weight.to(device)
    before = [t.clone() for t in pages]
    k = pool.randn((90, 3, 64)).to(device)
    for i in range(4):
        cu = torch.randint(-50, 200, (batch + 1,), generator=g).int()
        lens = torch.randint(-10, 60, (batch,), generator=g).int()
        K.paged_append(pages, table.to(device), lens.to(device), k, k, cu.to(device), weight=weight)
        K.paged_read(pages, table.to(device), lens.to(device), cu.to(device), 90)
    named = torch.zeros(300, dtype=torch.bool)
    named[table[(table >= 0) & (table < 300)].long()] = True
    for old, new in zip(before, pages):
        assert same(new[(~named).to(device)], old.cpu()[~named])
    assert same(weight[(~named).to(device)], pool.weight[~named])


# ------------------------------------------------------------------ attention over 4-bit rows

@pytest.mark.parametrize("lens, dim, heads, group, size", [
    ([1], 64, 1, 1, 16), ([0, 1, 15, 16, 17], 64, 2, 4, 16), ([33, 0, 700], 128, 2, 3, 32), ([513, 31], 256, 1, 8, 64),
    ([2100], 64, 2, 16, 16), ([5000, 3, 1200], 64, 1, 17, 64), ([2500, 900], 128, 2, 1, 256), ([4097], 256, 2, 2, 16),
    ([129, 128, 127, 64, 63, 65], 128, 3, 5, 128), ([0, 0], 64, 2, 2, 16), ([9000], 128, 1, 4, 32)])
def test_attention(device, lens, dim, heads, group, size):
    K = kernels()
    pool = B.Pool("e2m1", sum(-(-n // size) for n in lens) + 3, heads, size, dim, seed=sum(lens) + dim)
    table = pool.tables(lens)
    pool.poison(table, lens)
    q = pool.randn((len(lens), heads * group, dim))
    got = K.paged_attention(q.to(device), pool.pages(device), table.to(device), i32(lens, device), dim ** -0.5)
    R.check(got, *R.attention(pool, table, lens, q, dim ** -0.5))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_every_code_and_scale_attended(device, dim):
    """Values, then keys, of every byte of codes under every scale."""
    K = kernels()
    g = torch.Generator().manual_seed(dim)
    size, n = 16, 512
    codes = torch.randint(0, 256, (n // size, 1, size, dim // 2), generator=g).to(torch.uint8)
    scale = torch.arange(n * (dim // 16)).remainder(B.TOP + 1).to(torch.uint8).view(n // size, 1, size, dim // 16)
    key = torch.zeros_like(codes)  # codes 0: scores 0, all weights alike
    pool = B.Pool("e2m1", n // size, 1, size, dim, seed=1, bounds=False)
    pool.k, pool.k_scale, pool.v, pool.v_scale = key, torch.full_like(scale, 120), codes, scale
    table = torch.randperm(n // size, generator=g).int()[None].repeat(n, 1)
    q = torch.zeros((1, 1, dim), dtype=D16)
    q[0, 0, 0] = 100.0
    for i in range(n):
        page, row = int(table[0, i // size]), i % size
        pool.k[page, 0, row, 0] = 7 if i % 2 else 1  # 6 or 0.5 in the first coordinate
    for i in (0, 1, 17, 300, 511):
        got = K.paged_attention(q.to(device), pool.pages(device), table[:1].to(device), i32([i + 1], device), 1.0)
        R.check(got, *R.attention(pool, table[:1], [i + 1], q, 1.0), f"{dim} {i}")
    # keys of every code and scale, read by a query for each coordinate in turn
    pool.k, pool.k_scale = codes, scale.clamp_max(150)
    for c in range(0, dim, 7):
        q = torch.zeros((1, 1, dim), dtype=D16)
        q[0, 0, c] = 1.0
        got = K.paged_attention(q.to(device), pool.pages(device), table[:1].to(device), i32([n], device), 2.0 ** -6)
        R.check(got, *R.attention(pool, table[:1], [n], q, 2.0 ** -6), f"{dim} {c}")


@pytest.mark.parametrize("scale", [1e-3, 1.0, 30.0, -0.5, 0.0])
def test_scales_and_peaked_scores(device, scale):
    K = kernels()
    pool = B.Pool("e2m1", 130, 2, 16, 64, seed=9)
    lens = [2000, 7]
    table = pool.tables(lens)
    q = pool.randn((2, 8, 64), 2.0)
    got = K.paged_attention(q.to(device), pool.pages(device), table.to(device), i32(lens, device), scale)
    R.check(got, *R.attention(pool, table, lens, q, scale))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("where", ["k", "v", "both"])
def test_scales_that_are_no_numbers(device, dim, where):
    """A NaN key makes a head's result NaN; a NaN value that of its 16 coordinates."""
    K = kernels()
    pool = B.Pool("e2m1", 60, 2, 16, dim, seed=dim)
    lens = [600, 40, 300]
    table = pool.tables(lens)
    at = lambda b, t: (int(table[b, t // 16]), t % 16)
    if where != "v":
        page, row = at(0, 577)
        pool.k_scale[page, 1, row, 0] = 255
    if where != "k":
        page, row = at(2, 3)
        pool.v_scale[page, 0, row, dim // 16 - 1] = 255
        page, row = at(1, 39)
        pool.v_scale[page, 1, row] = 248  # infinite: zeros of it are NaN, other codes infinite
    q = pool.randn((3, 6, dim))
    got = K.paged_attention(q.to(device), pool.pages(device), table.to(device), i32(lens, device), 0.1)
    R.check(got, *R.attention(pool, table, lens, q, 0.1))


@pytest.mark.parametrize("dim, heads, group, size, count", [(64, 2, 4, 16, 20), (128, 1, 3, 64, 5), (256, 2, 1, 32, 9)])
def test_select_and_attend(device, dim, heads, group, size, count):
    K = kernels()
    lens = [30 * size + 5, size, 0, 3 * size]
    pool = B.Pool("e2m1", 70, heads, size, dim, seed=dim)
    table = pool.tables(lens)
    q = pool.randn((4, heads * group, dim))
    pages, t, n = pool.pages(device), table.to(device), i32(lens, device)
    chosen = K.page_select(q.to(device), pages, t, n, count)
    want = R.select(pool, table, lens, q, count, 1, 1)
    assert torch.equal(chosen.cpu(), want)
    got = K.paged_attention(q.to(device), pages, t, n, 0.125, chosen)
    R.check(got, *R.attention(pool, table, lens, q, 0.125, want))


def far_pool(kind, dim, heads, size, device):
    """A pool of over 2^32 bytes of codes and its last pages' numbers, with a small pool's rows in them."""
    small = B.Pool(kind, 40, heads, size, dim, seed=77)
    t = small.tensors()
    row = t["k"][0].numel() * t["k"].element_size()
    pages = (1 << 32) // row + 500
    far = {n: torch.zeros((pages, *x.shape[1:]), dtype=x.dtype, device=device) for n, x in t.items()}
    spots = torch.cat([torch.arange(20), torch.arange(pages - 20, pages)])
    for n, x in t.items():
        far[n].view(torch.uint8)[spots.to(device)] = x.to(device).view(torch.uint8)
    return small, far, spots.int()


@pytest.mark.parametrize("dim, size, heads", [(64, 16, 8), (256, 256, 2)])
def test_pools_past_32_bit_offsets(device, dim, size, heads):
    K = kernels()
    small, far, spots = far_pool("e2m1", dim, heads, size, device)
    lens = [12 * size - 3, 20 * size + 1]
    table = small.tables(lens)
    there = torch.where(table >= 0, spots[table.clamp_min(0).long()], -1)
    weight = far.pop("weight")
    pages = K.KVPages(**far)
    q = small.randn((2, 2 * heads, dim))
    got = K.paged_attention(q.to(device), pages, there.to(device), i32(lens, device), 0.1, weight=weight)
    want, tol = R.attention(small, table, lens, q, 0.1)
    R.check(got, want, tol)
    off = small.weigh(table, lens, q, 0.1)
    here = lambda: {n: x.view(torch.uint8)[spots.long().to(device)].view(x.dtype).cpu() for n, x in (far | {"weight": weight}).items()}
    assert ((here()["weight"].double() - small.weight).abs() <= off).all()
    small.weight = here()["weight"]
    new = K.paged_evict(pages, there.to(device), i32(lens, device), weight, 9 * size + 5, first=3, last=7)
    assert new.tolist() == small.evict(table, lens, 9 * size + 5, 3, 7)
    for n, x in here().items():
        assert same(x, getattr(small, n)), n
    k, v = small.randn((2, heads, dim)), small.randn((2, heads, dim))
    K.paged_append(pages, there.to(device), new, k.to(device), v.to(device), weight=weight)
    small.append(table, new.tolist(), k, v, [0, 1, 2])
    for n, x in here().items():
        assert same(x, getattr(small, n)), n
    assert int(sum((x.view(torch.uint8)[20:-20] != 0).any() for x in far.values())) == 0


# ------------------------------------------------------------------ accumulated weights

def weigh(device, pool, table, lens, q, scale, times=1):
    K = kernels()
    weight, pages = pool.weight.to(device), pool.pages(device)
    args = (q.to(device), pages, table.to(device), i32(lens, device), scale)
    want, tol = R.attention(pool, table, lens, q, scale)
    plain = K.paged_attention(*args)
    for _ in range(times):
        out = K.paged_attention(*args, weight=weight)
        off = pool.weigh(table, lens, q, scale)
    R.check(out, want, tol)
    assert same(out, plain.cpu())  # the same bits with and without
    got = weight.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(pool.weight))
    fine = ~torch.isnan(got)
    bad = ((got - pool.weight).abs() - times * off)[fine]
    assert float(bad.max()) <= 0, float(bad.max())
    return weight


@pytest.mark.parametrize("kind", B.KINDS)
@pytest.mark.parametrize("lens, dim, heads, group, size", [
    ([1], 64, 1, 1, 16), ([0, 1, 16, 37], 64, 2, 4, 16), ([2500, 900, 0], 128, 2, 3, 32), ([600, 31], 256, 1, 8, 64),
    ([3000], 64, 2, 17, 256), ([700] * 40, 64, 5, 1, 16), ([4097, 5], 256, 2, 2, 16)])
def test_weights(device, kind, lens, dim, heads, group, size):
    """Calls of one chunk and of several, in blocks of 4 waves and of many."""
    pool = B.Pool(kind, sum(-(-n // size) for n in lens) + 3, heads, size, dim, seed=sum(lens) + dim)
    table = pool.tables(lens)
    pool.poison(table, lens)
    q = pool.randn((len(lens), heads * group, dim))
    weigh(device, pool, table, lens, q, dim ** -0.5)


def test_weights_add_up(device):
    pool = B.Pool("e2m1", 90, 2, 16, 64, seed=3)
    lens = [700, 260]
    table = pool.tables(lens)
    weigh(device, pool, table, lens, pool.randn((2, 8, 64)), 0.3, times=3)


@pytest.mark.parametrize("kind", B.KINDS)
def test_weights_without_pages_and_numbers(device, kind):
    """Positions whose entry is no page, lengths past the table, scores that are NaN: nothing for the first, NaN on all positions of
    the last's head, and no word outside."""
    pool = B.Pool(kind, 60, 2, 16, 64, seed=4)
    lens = [2147483647, -5, 300, 160]
    table = torch.full((4, 20), -1, dtype=torch.int32)
    table[:, :] = torch.arange(80).view(4, 20)      # of the last sequence's entries none is a page
    table[0, 3], table[0, 7], table[2, 0] = -1, 99999, -7
    page = int(table[2, 5])
    if kind == "fp16":
        pool.k[page, 1, 3, 9] = math.nan
    elif kind == "e2m1":
        pool.k_scale[page, 1, 3, 2] = 255
    else:
        pool.k_scale[page, 1, 3] = math.nan
    got = weigh(device, pool, table, lens, pool.randn((4, 6, 64)), 0.1)
    assert torch.isnan(got).sum() == 19 * 16 - (320 - 300)  # every attended position of the third sequence's second head


def test_weights_of_scores_that_are_all_minus_infinite(device):
    pool = B.Pool("fp16", 30, 1, 16, 64, seed=4)
    lens = [200, 100]
    table = pool.tables(lens)
    q = torch.zeros((2, 2, 64), dtype=D16)
    q[:, :, 0] = 1.0
    pool.k[..., 0] = -math.inf
    pool.k[..., 1:] = 0.0
    for t in (3, 90):
        pool.k[int(table[1, t // 16]), 0, t % 16, 0] = 1.0
    weigh(device, pool, table, lens, q, 1.0)


# ------------------------------------------------------------------ eviction

def evict(device, pool, table, lens, keep, first, last):
    K = kernels()
    weight, pages = pool.weight.to(device), pool.pages(device)
    new = K.paged_evict(pages, table.to(device), i32(lens, device), weight, keep, first=first, last=last)
    assert new.tolist() == pool.evict(table, lens, keep, first, last)
    alike(pool, pages, weight)


@pytest.mark.parametrize("kind", B.KINDS)
@pytest.mark.parametrize("lens, dim, heads, size, keep, first, last", [
    ([2], 64, 1, 16, 1, 0, 0), ([2, 1], 64, 1, 16, 1, 1, 0), ([40, 17, 0, 16], 64, 2, 16, 16, 4, 5),
    ([300, 90, 120], 128, 3, 32, 100, 0, 0), ([300, 90, 120], 256, 2, 16, 111, 1, 110), ([700], 64, 8, 64, 699, 4, 64),
    ([500, 600], 128, 2, 256, 33, 33, 0), ([500, 600], 64, 2, 16, 33, 0, 33), ([1000, 20], 256, 1, 128, 513, 3, 100)])
def test_evict(device, kind, lens, dim, heads, size, keep, first, last):
    pool = B.Pool(kind, sum(-(-n // size) for n in lens) + 3, heads, size, dim, seed=keep + dim)
    table = pool.tables(lens)
    evict(device, pool, table, lens, keep, first, last)


def test_evict_without_bounds_and_of_many_sequences(device):
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(0, 60, (130,), generator=g).tolist()
    pool = B.Pool("e2m1", sum(-(-n // 16) for n in lens) + 1, 2, 16, 64, seed=8, bounds=False)
    evict(device, pool, pool.tables(lens), lens, 20, 1, 6)


@pytest.mark.parametrize("n, keep", [(9000, 4500), (20011, 300), (8200, 8199)])
def test_evict_long_sequences(device, n, keep):
    """More positions than a block holds the weights of."""
    pool = B.Pool("int8", -(-n // 256) + 1, 1, 256, 64, seed=n, bounds=False)
    pool.weight = torch.rand(pool.weight.shape, generator=pool.g)
    evict(device, pool, pool.tables([n]), [n], keep, 4, 64)


@pytest.mark.parametrize("n, keep, first, last", [(1000, 500, 4, 64), (16400, 5000, 3, 17), (35001, 20000, 7, 9), (35001, 70, 5, 1)])
def test_evict_by_weights_of_any_spread(device, n, keep, first, last):
    """Weights over all exponents, a step of fp32 apart, of few values, and alike but for some: the search for the last one
    kept takes from none to three histograms, or ends among 64."""
    g = torch.Generator().manual_seed(n + keep)
    size = 256
    P = -(-n // size)
    any_bits = torch.randint(0, 0x7f800000, (P * size,), generator=g, dtype=torch.int64).to(torch.int32).view(torch.float32)
    signed = any_bits * (torch.randint(0, 2, any_bits.shape, generator=g) * 2 - 1)
    steps = (torch.randint(0, 1 << 13, (P * size,), generator=g, dtype=torch.int32) + 0x3f800000).view(torch.float32)
    few = torch.randint(0, 3, (P * size,), generator=g).float()
    alike_but = torch.ones(P * size)
    alike_but[torch.randperm(n, generator=g)[:keep - first - last - 3]] = 1.0 + 2.0 ** -23
    for i, w in enumerate((any_bits, signed, steps, few, alike_but, torch.zeros(P * size), torch.rand(P * size, generator=g).log().neg())):
        pool = B.Pool("e2m1", P, 1, size, 64, seed=i, bounds=False)
        pool.weight = w.reshape(P, 1, size).clone()
        evict(device, pool, torch.arange(P, dtype=torch.int32).view(1, P), [n], keep, first, last)


def test_evict_ties_infinities_nan_and_missing_pages(device):
    """Ties go to the older position, NaN counts as infinite, a missing page's positions are given up first and
    move as zeros; what has no page is not written."""
    for kind in ("fp16", "e2m1"):
        pool = B.Pool(kind, 60, 2, 16, 64, seed=12)
        table = torch.arange(60, dtype=torch.int32).view(3, 20)
        table[0, 2], table[0, 11], table[1, 18] = -1, 77777, -1
        table[2, :15] = -1
        pool.weight[:20] = 1.0
        pool.weight[5, 0, 3:9], pool.weight[6, 1], pool.weight[21, 0], pool.weight[22, 1, 4] = math.nan, math.inf, -math.inf, -3.0
        pool.weight[30:35] = 0.0
        pool.weight[23, 0], pool.weight[24, 0] = -0.0, 0.0
        for keep, first, last in ((250, 0, 0), (100, 4, 10), (40, 0, 0)):
            evict(device, pool, table, [2147483647, 300, 320], keep, first, last)


def test_evict_leaves_short_sequences_and_other_pages_alone(device):
    K = kernels()
    pool = B.Pool("e4m3", 30, 2, 16, 64, seed=13)
    lens = [60, 100, 33]
    table = pool.tables(lens)
    pages, weight = pool.pages(device), pool.weight.to(device)
    for keep in (100, 101, 5000, 1 << 40):
        new = K.paged_evict(pages, table.to(device), i32(lens, device), weight, keep, first=4, last=64)
        assert new.tolist() == lens
        alike(pool, pages, weight)
    assert K.paged_evict(pages, table[:0].to(device), i32([], device), weight, 4, first=0, last=0).shape == (0,)
    none = torch.zeros((2, 0), dtype=torch.int32, device=device)
    assert K.paged_evict(pages, none, i32([5, 6], device), weight, 4, first=0, last=0).tolist() == [0, 0]
    alike(pool, pages, weight)


@pytest.mark.parametrize("kind", ["fp16", "e2m1"])
def test_strided_pools(device, kind):
    """K and V as parts of one allocation, pages apart, tables as part of a wider one."""
    K = kernels()
    pool = B.Pool(kind, 40, 2, 16, 64, seed=14)
    lens, keep = [200, 90], 70
    table = pool.tables(lens)
    joint = torch.zeros((40, 2, 3, *pool.k.shape[1:]), dtype=pool.k.dtype, device=device)
    joint[:, 0, 1], joint[:, 1, 1] = pool.k.to(device), pool.v.to(device)
    on = lambda t: None if t is None else t.to(device)
    pages = K.KVPages(joint[:, 0, 1], joint[:, 1, 1], on(pool.k_scale), on(pool.v_scale), on(pool.bounds))
    wide = torch.full((2, 40), 7, dtype=torch.int32, device=device)
    wide[:, 10:10 + table.shape[1]] = table.to(device)
    t, weight = wide[:, 10:10 + table.shape[1]], pool.weight.to(device)
    q = pool.randn((2, 6, 64))
    out = K.paged_attention(q.to(device), pages, t, i32(lens, device), 0.1, weight=weight)
    R.check(out, *R.attention(pool, table, lens, q, 0.1))
    pool.weight = weight.cpu()
    new = K.paged_evict(pages, t, i32(lens, device), weight, keep, first=2, last=8)
    assert new.tolist() == pool.evict(table, lens, keep, 2, 8)
    k = pool.randn((2, 2, 64))
    K.paged_append(pages, t, new, k.to(device), k.to(device), weight=weight)
    pool.append(table, new.tolist(), k, k, [0, 1, 2])
    alike(pool, pages, weight)
    joint[:, :, 1] = 0
    assert not joint.any()  # nothing between the pages


# ------------------------------------------------------------------ rotary positions

def turned(got, x, positions, inv_freq, layout, factor):
    """|error|: half a step of the result's type, and in fp32 the turn's error (cos and sin to 2^-23, two products and a sum
    of three roundings) times the pair; the angle's own error, 2^-53 of it, once for the product and once for the turns."""
    want = B.rotary(x.cpu(), positions.cpu(), inv_freq.cpu(), layout, factor)
    r = 2 * len(inv_freq)
    eps = torch.finfo(x.dtype).eps / 2
    y = x.cpu().double()
    a, b = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    pair = torch.zeros_like(y)
    pair[..., a] = pair[..., b] = (y[..., a].abs() + y[..., b].abs()) * abs(factor)
    angle = float((positions.double().abs().max() * inv_freq.abs().max()).cpu()) if len(positions) else 0.0
    tol = want.abs() * eps + pair * (5 * 2.0 ** -24 + 4 * angle * 2.0 ** -53) + torch.finfo(x.dtype).tiny * eps * 2
    assert got.dtype == x.dtype and got.shape == x.shape
    off = (got.cpu().double() - want).abs() - tol
    assert float(off.max()) <= 0, float((got.cpu().double() - want).abs().max())
    if r < x.shape[2]:
        assert torch.equal(got[..., r:], x[..., r:])


def freq(r, device, theta=500000.0):
    return (theta ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)).to(device)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows, q_heads, kv_heads, dim, r", [
    (1, 32, 4, 64, 64), (33, 8, 2, 64, 32), (7, 3, 1, 128, 128), (129, 4, 4, 128, 64), (5, 2, 1, 256, 256), (1000, 8, 8, 64, 64),
    (3, 1, 1, 80, 20), (4, 5, 2, 96, 96), (17, 2, 2, 64, 2), (9, 6, 3, 64, 62), (2, 1, 1, 2, 2), (6, 2, 1, 7, 6), (3, 2, 1, 1024, 1024),
    (300, 40, 40, 128, 128), (4100, 2, 1, 64, 48)])
def test_rotary(device, dtype, layout, rows, q_heads, kv_heads, dim, r):
    """New tensors from parts of a projection's output, and the same in place; queries alone."""
    K = kernels()
    g = torch.Generator().manual_seed(rows + dim)
    wide = torch.randn((rows, q_heads + 2 * kv_heads, dim), generator=g).to(dtype).to(device)
    q, k = wide[:, :q_heads], wide[:, q_heads:q_heads + kv_heads]
    pos = torch.randint(0, 131072, (rows,), generator=g).int().to(device)
    f = freq(r, device)
    qo, ko = K.rotary(q, k, pos, f, layout=layout, factor=1.25)
    turned(qo, q, pos, f, layout, 1.25)
    turned(ko, k, pos, f, layout, 1.25)
    alone, none = K.rotary(q, None, pos.long(), f, layout=layout, factor=1.25)
    assert none is None and torch.equal(alone, qo)
    before = wide.clone()
    q2, k2 = K.rotary(q, k, pos, f, layout=layout, factor=1.25, inplace=True)
    assert q2 is q and k2 is k and torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(wide[:, q_heads + kv_heads:], before[:, q_heads + kv_heads:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_strides(device, layout):
    """Heads before rows, rows that are far apart, odd offsets, coordinates that are not dense."""
    K = kernels()
    g = torch.Generator().manual_seed(2)
    pos, f = torch.arange(50, device=device, dtype=torch.int32) * 7, freq(64, device)
    base = torch.randn(50 * 8 * 64 * 3 + 9, generator=g).half().to(device)
    for off, shape, strides in ((0, (50, 8, 64), (64, 50 * 64, 1)), (8, (50, 8, 64), (8 * 64 * 3, 64, 1)),
                                (1, (50, 8, 64), (8 * 64, 64, 1)), (3, (50, 8, 64), (8 * 67, 67, 1)), (0, (50, 8, 64), (8 * 64 * 2, 128, 2))):
        x = base.as_strided(shape, strides, off)
        keep = base.clone()
        got, other = K.rotary(x, x[:, :3], pos, f, layout=layout)
        turned(got, x, pos, f, layout, 1.0)
        assert torch.equal(other, got[:, :3]) and torch.equal(base, keep)
        if strides[2] == 1:
            K.rotary(x, None, pos, f, layout=layout, inplace=True)
            assert torch.equal(x, got)
            untouched = torch.ones_like(base, dtype=torch.bool)
            untouched.as_strided(shape, strides, off).fill_(False)
            assert torch.equal(base[untouched], keep[untouched])
            base.copy_(keep)


def test_rotary_far_and_negative_positions(device):
    """Positions up to a billion: the angle's turns are counted in 64 bits."""
    K = kernels()
    g = torch.Generator().manual_seed(3)
    x = torch.randn((40, 2, 64), generator=g).to(device)
    for far in (0, -1, 1 << 20, 10 ** 9, 2 ** 31 - 1, -(2 ** 31)):
        pos = torch.full((40,), far, dtype=torch.int64).to(device)
        f = freq(64, device)
        f[0] = 1.0
        turned(K.rotary(x, None, pos, f)[0], x, pos, f, "half", 1.0)
    same_turn = K.rotary(x, None, torch.zeros(40, dtype=torch.int32, device=device), freq(64, device))[0]
    assert torch.equal(same_turn, x)  # position 0 turns nothing


def test_rotary_quarters(device):
    """Turns at and near every eighth of a circle."""
    K = kernels()
    f = (torch.arange(-20, 21, dtype=torch.float64) * math.pi / 4).to(device)
    f = torch.cat([f, f + 1e-9, f - 1e-9])
    g = torch.Generator().manual_seed(4)
    x = torch.randn((3, 2, 2 * len(f)), generator=g).to(device)
    pos = torch.tensor([1, 2, 3], dtype=torch.int32, device=device)
    turned(K.rotary(x, None, pos, f)[0], x, pos, f, "half", 1.0)


def test_rotary_infinities_and_empty_calls(device):
    K = kernels()
    f = freq(64, device)
    x = torch.ones((2, 2, 64), dtype=D16, device=device)
    x[0, 0, 3], x[1, 1, 40] = math.inf, math.nan
    got = K.rotary(x, None, i32([5, 6], device), f)[0]
    bad = ~torch.isfinite(got)
    assert bad[0, 0, 3] and bad[0, 0, 35] and bad[1, 1, 8] and bad[1, 1, 40] and int(bad.sum()) == 4
    none = torch.zeros((0, 2, 64), dtype=D16, device=device)
    assert K.rotary(none, none, i32([], device), f)[0].shape == (0, 2, 64)
    q, k = K.rotary(x[:, :0], x, i32([5, 6], device), f)
    assert q.shape == (2, 0, 64) and same(k, got.cpu())
    q, k = K.rotary(x, x[:, :0], i32([5, 6], device), f)
    assert k.shape == (2, 0, 64) and same(q, got.cpu())


def test_rotary_of_the_llama_layer(device):
    """The layer's own tables give the same turns."""
    from apple_amd.layer import LLAMA3_ROPE_SCALING, rope_cos_sin, rope_inv_freq

    K = kernels()
    g = torch.Generator().manual_seed(6)
    x = torch.randn((20, 4, 64), generator=g).half().to(device)
    pos = torch.arange(8180, 8200, device=device)
    cos, sin = rope_cos_sin(pos, 64, 500000.0, LLAMA3_ROPE_SCALING)
    f = rope_inv_freq(64, 500000.0, LLAMA3_ROPE_SCALING, device)
    xf = x.float()
    want = (xf * cos[:, None] + torch.cat([-xf[..., 32:], xf[..., :32]], -1) * sin[:, None]).half()
    got = K.rotary(x, None, pos, f)[0]
    # either is off by half a step of fp16 at most, but for fp32's own errors
    assert ((got - want).abs().float() <= want.abs().float() * 2.0 ** -10 + 2.0 ** -22).all()


# ------------------------------------------------------------------ calls

def test_other_streams(device):
    """Every call on a stream of the program's own, two at once."""
    K = kernels()
    pools = [B.Pool("e2m1", 120, 2, 16, 64, seed=45 + i) for i in range(2)]
    lens = [1700]
    runs = []
    for pool in pools:
        table = pool.tables(lens)
        runs.append((pool, table, pool.randn((1, 8, 64)), pool.pages(device), table.to(device), i32(lens, device), pool.weight.to(device)))
    streams = [torch.cuda.Stream() for _ in runs]
    got = []
    for s, (pool, _, q, pages, t, n, w) in zip(streams, runs):
        qd, f = q.to(device), freq(64, device)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            turned_q, _ = K.rotary(qd, None, n, f)
            out = K.paged_attention(turned_q, pages, t, n, 0.125, weight=w)
            before = w.clone()
            new = K.paged_evict(pages, t, n, w, 500, first=4, last=64)
        got.append((turned_q, out, before, new, w))
    torch.cuda.synchronize()
    for (pool, table, q, pages, *_), (turned_q, out, before, new, w) in zip(runs, got):
        R.check(out, *R.attention(pool, table, lens, turned_q.cpu(), 0.125))
        pool.weight = before.cpu()
        assert new.tolist() == pool.evict(table, lens, 500, 4, 64)
        alike(pool, pages, w)


def test_captured_steps(device):
    """A step in a graph, rotary to weights, among the program's own work; an eviction in another; replays follow the device's state."""
    K = kernels()
    H, size, start, keep = 2, 16, [5, 0, 900], 800
    pool = B.Pool("e2m1", 160, H, size, 64, seed=50)
    table = pool.tables([n + 60 for n in start])
    pages, weight, t, lens = pool.pages(device), pool.weight.to(device), table.to(device), i32(start, device)
    pos, f = i32(start, device), freq(64, device)
    k, v, q = (torch.zeros((3, n, 64), dtype=D16, device=device) for n in (H, H, 8))

    def step():
        qr, kr = K.rotary(q, k, pos, f)
        K.paged_append(pages, t, lens, kr, v, weight=weight)
        lens.add_(1)
        pos.add_(1)
        return qr, kr, K.paged_attention(qr, pages, t, lens, 0.125, weight=weight)

    def cut():
        lens.copy_(K.paged_evict(pages, t, lens, weight, keep, first=4, last=100))

    state = list(pages) + [weight, lens, pos]
    keep_state = [x.clone() for x in state]
    step()
    cut()
    graphs, outs = [], []
    for call in (step, cut):
        for x, y in zip(state, keep_state):
            x.copy_(y)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for x, y in zip(state, keep_state):
        x.copy_(y)
    qr, kr, out = outs[0]
    now, at = list(start), list(start)
    for i in range(12):
        rows = [pool.randn((3, n, 64)) for n in (H, H, 8)]
        for x, r in zip((k, v, q), rows):
            x.copy_(r)
        graphs[0].replay()
        p = torch.tensor(at)
        turned(qr, rows[2].to(device), p.to(device), f, "half", 1.0)
        turned(kr, rows[0].to(device), p.to(device), f, "half", 1.0)
        pool.append(table, now, kr.cpu(), rows[1], [0, 1, 2, 3])
        now, at = [n + 1 for n in now], [n + 1 for n in at]
        off = pool.weigh(table, now, qr.cpu(), 0.125)
        assert ((weight.cpu().double() - pool.weight).abs() <= off).all(), i
        pool.weight = weight.cpu()
        R.check(out, *R.attention(pool, table, now, qr.cpu(), 0.125), f"replay {i}")
        torch.zeros(1 << 20, device=device).sum().item()  # the program's own work between replays
        if i % 4 == 1:
            graphs[1].replay()
            now = pool.evict(table, now, keep, 4, 100)
            alike(pool, pages, weight)
        assert lens.tolist() == now and pos.tolist() == at


def test_wrappers_refuse(device):
    K = kernels()
    pool = B.Pool("e2m1", 8, 2, 16, 64, seed=60)
    pages, t, n, w = pool.pages(device), torch.zeros((2, 4), dtype=torch.int32, device=device), i32([5, 6], device), pool.weight.to(device)
    q = torch.zeros((2, 4, 64), dtype=D16, device=device)
    rows, f, p = q[:, :2].contiguous(), freq(64, device), i32([1, 2], device)
    s8 = torch.zeros((8, 2, 16), device=device)
    grad = q.float().requires_grad_()
    bad = [
        lambda: K.paged_attention(q, pages._replace(k_scale=s8, v_scale=s8), t, n, 0.1),
        lambda: K.paged_attention(q, pages._replace(k_scale=None), t, n, 0.1),
        lambda: K.paged_attention(q[..., :32].contiguous(), pages, t, n, 0.1),
        lambda: K.paged_attention(q, pages._replace(k=pages.k[..., :16], v=pages.v[..., :16]), t, n, 0.1),
        lambda: K.paged_append(pages, t, n, rows[..., :32], rows[..., :32]),
        lambda: K.paged_append(pages, t, n, rows, rows, weight=w.half()), lambda: K.paged_append(pages, t, n, rows, rows, weight=w[:4]),
        lambda: K.paged_append(pages, t, n, rows, rows, weight=w.cpu()),
        lambda: K.paged_attention(q, pages, t, n, 0.1, weight=w.transpose(1, 2)),
        lambda: K.paged_attention(q, pages, t, n, 0.1, torch.zeros((2, 2, 3), dtype=torch.int32, device=device), weight=w),
        lambda: K.paged_evict(pages, t, n, None, 4), lambda: K.paged_evict(pages, t, n, w.double(), 4, first=0, last=0),
        lambda: K.paged_evict(pages, t, n, w, 0, first=0, last=0), lambda: K.paged_evict(pages, t, n, w, 4),
        lambda: K.paged_evict(pages, t, n, w, 4, first=-1, last=0), lambda: K.paged_evict(pages, t, n.long(), w, 4, first=0, last=0),
        lambda: K.rotary(q[0], None, p, f), lambda: K.rotary(q.double(), None, p, f), lambda: K.rotary(q, rows.float(), p, f),
        lambda: K.rotary(q, rows[:1], p, f), lambda: K.rotary(q, rows[..., :32], p, f), lambda: K.rotary(q, None, p[:1], f),
        lambda: K.rotary(q, None, p.float(), f), lambda: K.rotary(q, None, p.cpu(), f), lambda: K.rotary(q, None, p, f.float()),
        lambda: K.rotary(q, None, p, freq(66, device)), lambda: K.rotary(q, None, p, f[:0]), lambda: K.rotary(q, None, p, f.cpu()),
        lambda: K.rotary(q, None, p, f, layout="rows"), lambda: K.rotary(q, q, p, f, inplace=True),
        lambda: K.rotary(q[:1].expand(2, 4, 64), None, p, f, inplace=True), lambda: K.rotary(q[..., ::2], None, p, f[:8], inplace=True),
        lambda: K.rotary(grad, None, p, f), lambda: K.rotary(torch.zeros((2, 1, 2000), device=device), None, p, f)]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was accepted")
    with torch.no_grad():
        K.rotary(grad, None, p, f)


# ------------------------------------------------------------------ the cache

def test_calls_that_would_lose_gradients_or_race_are_refused(device):
    K = kernels()
    pool = B.Pool("fp16", 8, 2, 16, 64, seed=61)
    pages, n, w = pool.pages(device), i32([5, 6], device), pool.weight.to(device)
    q = torch.zeros((2, 4, 64), dtype=D16, device=device)
    one = torch.zeros((1, 4), dtype=torch.int32, device=device)
    with pytest.raises(RuntimeError, match="no gradients"):
        K.rotary(q, None, i32([1, 2], device), freq(64, device).requires_grad_())
    with torch.no_grad():
        K.rotary(q, None, i32([1, 2], device), freq(64, device).requires_grad_())
    with pytest.raises(ValueError, match="share a table"):
        K.paged_attention(q, pages, one.expand(2, 4), n, 0.1, weight=w)
    with pytest.raises(ValueError, match="share a table"):
        K.paged_evict(pages, one.expand(2, 4), n, w, 4, first=0, last=0)
    K.paged_attention(q, pages, one.expand(2, 4), n, 0.1)  # read alone they may
    K.paged_attention(q[:1], pages, one, n[:1], 0.1, weight=w)


@pytest.mark.parametrize("kind, dim, size", [("e2m1", 64, 16), ("e2m1", 128, 32), ("fp16", 64, 16), ("int8", 256, 16)])
def test_cache_in_bounded_memory(device, kind, dim, size):
    """Prompts, steps with rotary positions, evictions, a sequence that ends and one that takes its place."""
    from apple_amd.paged import RFSNPagedKVCache
    from apple_amd.storage import RFSNConfig

    cfg = RFSNConfig(hidden_dim=8 * dim, num_heads=8, num_kv_heads=2, head_dim=dim, num_subspaces=8, subspace_dim=dim // 8)
    cache = RFSNPagedKVCache(cfg, batch=3, pages=1600 // size, page_size=size, page_type=kind, device=device, weights=True)
    g = torch.Generator().manual_seed(dim)
    rand = lambda *s: torch.randn(s, generator=g).half()
    model = B.Pool(kind, 1600 // size, 2, size, dim, seed=1)
    f = freq(dim, device)
    held, given = [0] * 3, [0] * 3

    def pool_now():
        for name, t in cache.pages._asdict().items():
            if t is not None:
                setattr(model, name, t.cpu())
        model.weight = cache.weight.cpu()
        assert cache.num_tokens == held == cache.lens.tolist()
        return cache.table.cpu()

    def append(counts):
        each = counts or [1, 1, 1]
        n = sum(each)
        q, k, v = rand(n, 8, dim), rand(n, 2, dim), rand(n, 2, dim)
        pos = torch.tensor([a + i for a, c in zip(given, each) for i in range(c)])
        qr, kr = cache.rotary(q.to(device), k.to(device), f, counts, layout="interleaved")
        turned(qr, q.to(device), pos.to(device), f, "interleaved", 1.0)
        turned(kr, k.to(device), pos.to(device), f, "interleaved", 1.0)
        pool_now()
        cache.append(kr, v.to(device), counts)
        model.append(cache.table.cpu(), held, kr.cpu(), v, CU(each))
        for b, c in enumerate(each):
            held[b] += c
            given[b] += c
        alike(model, cache.pages, cache.weight)
        return qr

    def attend(q):
        t = pool_now()
        got = cache.attention_forward(q)
        R.check(got, *R.attention(model, t, held, q.cpu(), dim ** -0.5))
        off = model.weigh(t, held, q.cpu(), dim ** -0.5)
        assert ((cache.weight.cpu().double() - model.weight).abs() <= off).all()

    append([300, 0, 120])
    append([0, 417, 3])
    for i in range(40):
        q = append(None)
        if i % 3 == 0:
            attend(q)
        if i in (10, 25):
            t = pool_now()
            held[:] = model.evict(t, held, 200, 4, 50)
            cache.evict(200, 4, 50)
            alike(model, cache.pages, cache.weight)
            assert cache.free_pages == 1600 // size - sum(-(-n // size) for n in held)
    q = rand(20, 8, dim)
    out = cache.prompt_attention(0, q.to(device))
    t = pool_now()
    for i in (0, 19):
        want, tol = R.attention(model, t[:1], [held[0] - 19 + i], q[i:i + 1], dim ** -0.5)
        R.check(out[i:i + 1], want, tol + 2.0 ** -10 * want.abs().amax())  # rows as fp16, its own kernel's steps
    with pytest.raises(ValueError, match="gap"):
        cache.prompt_attention(0, rand(100, 8, dim).to(device))
    want = R.select(model, t, held, q[:3], 4, 1, 1)
    before = cache.weight.clone()
    R.check(cache.attention_forward(q[:3].to(device), sparse_pages=4), *R.attention(model, t, held, q[:3], dim ** -0.5, want))
    assert torch.equal(before, cache.weight)
    cache.release(1)
    held[1] = given[1] = 0
    attend(rand(3, 8, dim).to(device))
    append([0, 40, 0])
    attend(append(None))
