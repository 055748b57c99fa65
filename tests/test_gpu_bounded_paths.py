"""A paged cache in bounded memory on the GPU, where other calls than test_gpu_bounded.py's lead: in-place results among
a program's gradients, and the kernels' variants for large calls, against 64 bits."""

import math
import random

import pytest
import torch

from tests import bounded_reference as B
from tests import paged_reference as R
from tests.test_gpu_bounded import freq, i32, kernels, turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["q", "k"])
def test_rotary_in_place_is_seen_by_autograd(device, which):
    """A product whose gradient needs the rows as they were: as with torch's own in-place operators, its backward pass is
    refused, views of the rows included, and rows that nothing watches are turned as before."""
    K = kernels()
    pos, f = i32([3, 9, 4], device), freq(64, device)
    wide = torch.randn((3, 6, 64), device=device)
    q, k = wide[:, :4], wide[:, 4:]
    w = torch.ones(64, device=device, requires_grad=True)
    y = (q if which == "q" else k) * w
    before = wide.clone()
    K.rotary(q, k, pos, f, inplace=True)
    turned(q, before[:, :4], pos, f, "half", 1.0)
    turned(k, before[:, 4:], pos, f, "half", 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    other = torch.randn((3, 4, 64), device=device)
    y = other * w
    K.rotary(other, None, pos, f)  # new tensors: nothing was changed
    y.sum().backward()
    # 12 terms: 11 roundings of at most half a step of the sum of magnitudes on either side
    assert ((w.grad - other.sum((0, 1))).abs() <= 22 * 2.0 ** -24 * other.abs().sum((0, 1))).all()


def test_a_batch_attended_in_parts(device, monkeypatch):
    """Scores that may not pass the pool's rows: a long sequence among short and empty ones, weights and results as in one call,
    in no more memory."""
    from apple_amd import paged
    from apple_amd.storage import RFSNConfig

    lens, dim, size = [40, 0, 1700, 16, 0, 33, 700, 5], 64, 16
    cfg = RFSNConfig(hidden_dim=8 * dim, num_heads=8, num_kv_heads=2, head_dim=dim, num_subspaces=8, subspace_dim=dim // 8)
    held = sum(-(-n // size) for n in lens)
    cache = paged.RFSNPagedKVCache(cfg, batch=8, pages=held, page_size=size, page_type="e2m1", device=device, weights=True)
    model = B.Pool("e2m1", held, 2, size, dim, seed=1)
    k, v, q = (model.randn((n, h, dim)) for n, h in ((sum(lens), 2), (sum(lens), 2), (8, 8)))
    cache.append(k.to(device), v.to(device), lens)
    for name, t in cache.pages._asdict().items():
        setattr(model, name, t.cpu())
    model.weight = cache.weight.cpu()
    table, qd = cache.table.cpu(), q.to(device)
    used = []
    for least in (paged.SCORES_AT_LEAST, 0):
        monkeypatch.setattr(paged, "SCORES_AT_LEAST", least)
        cache.weight.zero_()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = cache.attention_forward(qd)
        used.append(torch.cuda.max_memory_allocated() - before)
        R.check(out, *R.attention(model, table, lens, q, dim ** -0.5))
        model.weight = torch.zeros_like(cache.weight.cpu())
        off = model.weigh(table, lens, q, dim ** -0.5)
        assert ((cache.weight.cpu().double() - model.weight).abs() <= off).all()
    assert used[0] >= 8 * 8 * 107 * size * 4  # batch x longest
    assert used[1] < held * size * 8 * 4 + (64 << 10), used  # the pool's rows, partial results and the allocator's steps


# ------------------------------------------------------------------ attention and weights in blocks of four waves, and of long calls

def some(seed, batch, most, *first):
    """Lengths 0 to most, the first of them given."""
    rng = random.Random(seed)
    return list(first) + [rng.randrange(most + 1) for _ in range(batch - len(first))]


# KV heads, query heads of each, page size, lengths, positions that the table has room for, and which of the kernels' variants
# that is (test_bounded_rules.py holds the host's plan to it): blocks of many waves, loads past the caches, chunks
# cut by the lengths.  `dims`: head sizes.
CALLS = {
    "four_waves": dict(kv=8, group=4, size=16, lens=[9000, 300, 0, 2500], room=16000, dims=(64, 128), wide=0, once=0, cut=1),
    # one chunk a sequence, so the attention's blocks have the whole sums
    "four_waves_uncut": dict(kv=4, group=2, size=16, lens=some(1, 300, 512, 512, 0, 1), room=512, dims=(64, 128), wide=0, once=0, cut=0),
    # more pages than the last-level cache has room for, the sequences' scattered among them
    "past_the_caches": dict(kv=4, group=3, size=16, lens=[3000, 0, 17, 555], room=0, dims=(64, 128, 256), wide=0, once=1, cut=1),
    # batches that fill the chip by themselves: 4-bit rows of 128 are weighed in more chunks than sequences
    "full": dict(kv=32, group=1, size=64, lens=some(2, 24, 900, 4000), room=4200, dims=(64, 128), wide=0, once=0, cut=1),
    # a wave takes more tiles than it looks pages up for at once; 64 query heads' sums are held at a time
    "many_tiles": dict(kv=1, group=1024, size=64, lens=[80000], room=80000, dims=(64,), wide=0, once=0, cut=1),
    # more than 64 chunks of one sequence, few rows of results and many
    "many_chunks": dict(kv=1, group=1, size=16, lens=[40001], room=40001, dims=(64,), wide=1, once=0, cut=1),
    "many_chunks_of_many_heads": dict(kv=4, group=8, size=16, lens=some(3, 9, 300, 40000), room=40000, dims=(64,), wide=0, once=0, cut=1),
    # blocks of the weights' launch that take a second 1,024 positions of their sequence, rows joined by 4 and by 16 waves
    "second_round": dict(kv=8, group=2, size=16, lens=some(4, 32, 400, 20000, 16385), room=20000, dims=(64,), wide=0, once=0, cut=1),
    "second_round_16": dict(kv=8, group=1, size=16, lens=some(5, 32, 400, 20000, 16384), room=20000, dims=(64,), wide=0, once=0, cut=1),
    "second_round_many_heads": dict(kv=16, group=70, size=16, lens=some(6, 16, 200, 17500), room=17500, dims=(64,), wide=0, once=0, cut=1),
    "many_heads": dict(kv=1, group=71, size=16, lens=[700, 0, 33, 1990], room=2000, dims=(64,), wide=1, once=0, cut=1),
    "more_heads": dict(kv=2, group=130, size=16, lens=[1500, 17, 1999], room=2000, dims=(64, 256), wide=1, once=0, cut=1),
}
ROW = {"fp16": 4.0, "int8": 2.0, "e4m3": 2.0, "e2m1": 1.125}  # bytes of K and V per coordinate


def shape_of(call, kind, dim):
    """(pages of the pool, table's width): for `once` 256 MiB of pages and a table with room for them."""
    c = CALLS[call]
    need = sum(-(-n // c["size"]) for n in c["lens"])
    if not c["once"]:
        return need + 3, -(-c["room"] // c["size"])
    pages = math.ceil((256 << 20) / (ROW[kind] * dim * c["kv"] * c["size"])) + 50
    return pages, -(-pages // len(c["lens"])) + 1


class DevicePool:
    """A pool on the device, garbage (NaN, where its type has it) in all rows that no sequence holds."""

    def __init__(self, device, kind, dim, call, seed):
        K = kernels()
        c = CALLS[call]
        self.kind, self.size, self.heads, self.dim = kind, c["size"], c["kv"], dim
        pages, width = shape_of(call, kind, dim)
        g = torch.Generator(device=device).manual_seed(seed)
        lens = c["lens"]
        order = torch.randperm(pages, generator=g, device=device).int()
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32, device=device)
        self.held = torch.zeros((pages, self.size), dtype=torch.bool, device=device)
        at = 0
        for b, n in enumerate(lens):
            need = -(-n // self.size)
            self.table[b, :need] = order[at:at + need]
            full = torch.arange(need * self.size, device=device).view(need, self.size) < n
            self.held[order[at:at + need].long()] = full
            at += need
        shape = (pages, self.heads, self.size, dim)
        free = (~self.held)[:, None, :].expand(-1, self.heads, -1)
        randn = lambda *s: torch.randn(s, generator=g, device=device)
        rows, scales = [], []
        for _ in range(2):
            if kind == "fp16":
                x = torch.empty(shape, dtype=torch.float16, device=device).normal_(generator=g)
                x[free] = math.nan
                rows.append(x)
                continue
            if kind == "e2m1":
                rows.append(torch.randint(0, 256, (*shape[:3], dim // 2), generator=g, dtype=torch.uint8, device=device))
                s = torch.randint(96, 110, (*shape[:3], dim // 16), generator=g, dtype=torch.uint8, device=device)  # 1/8 to 0.4
                s[free] = 255
            else:
                if kind == "int8":
                    x = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, device=device)
                else:
                    x = (randn(*shape) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
                s = (randn(*shape[:3]).abs() + 0.1) / 100
                s[free] = math.nan
                rows.append(x)
            scales.append(s)
        self.pages = K.KVPages(*rows, *(scales or (None, None)))
        self.weight = randn(pages, self.heads, self.size).abs()
        self.weight[free] = math.nan
        self.q = (randn(len(lens), c["kv"] * c["group"], dim) * (1.0 if dim < 256 else 0.7)).half()
        self.lens = torch.tensor(lens, dtype=torch.int32, device=device)

    def place(self, b):
        n = int(self.lens[b])
        t = torch.arange(n, device=self.table.device)
        return self.table[b].long()[t // self.size], t % self.size

    def rows(self, b, name):
        """K or V of sequence b, [H, n, D] in 64 bits."""
        page, row = self.place(b)
        x = getattr(self.pages, name)[page, :, row]
        if self.kind == "fp16":
            return x.double().transpose(0, 1).contiguous()
        s = getattr(self.pages, name + "_scale")[page, :, row]
        if self.kind == "e2m1":
            value = torch.cat([B.MAGNITUDES, -B.MAGNITUDES]).to(x.device)
            c = torch.stack([x & 15, x >> 4], -1).flatten(-2).long()
            v = value[c].unflatten(-1, (-1, 16)) * B.SCALES.to(x.device)[s.long()][..., None]
            return v.flatten(-2).transpose(0, 1).contiguous()
        return (x.float().double() * s.double()[..., None]).transpose(0, 1).contiguous()

    def check(self, out, weight, scale):
        """Results and weights against 64 bits, a sequence at a time, with the tolerances of paged_reference.attention and
        bounded_reference.Pool.weigh; rows that no sequence holds keep their weight."""
        G = self.q.shape[1] // self.heads
        for b in range(len(self.lens)):
            page, row = self.place(b)
            n = len(page)
            if n == 0:
                assert not out[b].any()
                continue
            k, v = self.rows(b, "k"), self.rows(b, "v")
            was = self.weight[page, :, row].double().t()
            got = weight[page, :, row].double().t()
            for h in range(self.heads):
                q = self.q[b, h * G:(h + 1) * G].double()
                s = (q @ k[h].t().contiguous()) * scale
                size = ((q.abs() @ k[h].abs().t().contiguous()) * abs(scale)).nan_to_num(0, 0, 0).amax(-1)
                p = torch.softmax(s, -1)
                p = torch.where(p < 2.0 ** -149, 0.0, p)
                want = (p @ v[h])
                big = float(v[h].abs().nan_to_num(0, 0, 0).amax())
                tol = want.abs().nan_to_num(0, 0, 0) * 2.0 ** -11 + 2.0 ** -25 + big * (
                    2 * (self.dim + 4) * 2.0 ** -24 * size[:, None] + 2 * n * 2.0 ** -24 + 2.0 ** -16)
                R.check(out[b, h * G:(h + 1) * G], want.cpu(), tol.cpu(), f"sequence {b} head {h}")
                total = was[h] + p.sum(0)
                off = (p.nan_to_num(0) * (2 * (self.dim + 4) * size[:, None] + n + 16) * 2.0 ** -24 + 2.0 ** -126).sum(0)
                off += total.abs().nan_to_num(0) * (G + 1) * 2.0 ** -24
                assert torch.equal(torch.isnan(got[h]), torch.isnan(total)), (b, h)
                bad = ((got[h] - total).abs() - off).nan_to_num(0)
                assert float(bad.amax()) <= 0, (b, h, int(bad.argmax()), float(bad.amax()))
        free = ~self.held
        assert torch.isnan(weight.transpose(1, 2)[free]).all()


def attend_and_weigh(pool, scale):
    K = kernels()
    args = (pool.q, pool.pages, pool.table, pool.lens, scale)
    plain = K.paged_attention(*args)
    weight = pool.weight.clone()
    out = K.paged_attention(*args, weight=weight)
    assert ((out == plain) | (torch.isnan(out) & torch.isnan(plain))).all()  # the same bits with and without
    pool.check(out, weight, scale)


@pytest.mark.parametrize("call, kind, dim", [
    (call, kind, dim) for call, c in CALLS.items() for dim in c["dims"]
    for kind in (B.KINDS if call.startswith(("four", "past")) else ("fp16", "e2m1"))])
def test_results_and_weights(device, call, kind, dim):
    attend_and_weigh(DevicePool(device, kind, dim, call, seed=dim + len(call)), dim ** -0.5)


@pytest.mark.parametrize("kind", B.KINDS)
@pytest.mark.parametrize("call, dim", [("four_waves", 64), ("four_waves", 128), ("past_the_caches", 64), ("past_the_caches", 256)])
def test_no_numbers_in_blocks_of_four_waves(device, call, kind, dim):
    """A NaN key makes a head's results and weights NaN, a NaN value results alone."""
    pool = DevicePool(device, kind, dim, call, seed=3)
    page, row = (x[-200] for x in pool.place(0))
    x = pool.pages.k if kind == "fp16" else pool.pages.k_scale
    x[page, 1, row] = 255 if kind == "e2m1" else math.nan
    page, row = (x[9] for x in pool.place(3))
    x = pool.pages.v if kind == "fp16" else pool.pages.v_scale
    x[page, 0, row] = 255 if kind == "e2m1" else math.nan
    attend_and_weigh(pool, dim ** -0.5)


@pytest.mark.parametrize("scale", [3.0, -0.4])
def test_peaked_scores_in_blocks_of_four_waves(device, scale):
    """Maxima that move, weights that vanish, and a scale that turns the order."""
    for kind in ("fp16", "e2m1"):
        attend_and_weigh(DevicePool(device, kind, 128, "four_waves", seed=4), scale)


@pytest.mark.parametrize("dim", [64, 128])
def test_chosen_pages_in_chunks_of_many_tiles(device, dim):
    """4-bit pages of a list, so many of them that a wave looks its pages up more than once (4,096 query heads fill the
    chip, so a chunk has a fourth of the list: over 32 tiles of 32 positions for each of 4 waves)."""
    K = kernels()
    pool = DevicePool(device, "e2m1", dim, "many_tiles", seed=dim)
    width, count = pool.table.shape[1], 330
    g = torch.Generator().manual_seed(dim)
    chosen = torch.randperm(width - 1, generator=g)[:count - 1].sort().values.int()
    chosen = torch.cat([chosen, torch.tensor([width - 1], dtype=torch.int32)]).view(1, 1, count).to(device)
    q = torch.randn((1, 4096, dim), generator=g).half().to(device)
    out = K.paged_attention(q, pool.pages, pool.table, pool.lens, dim ** -0.5, chosen)
    k, v = pool.rows(0, "k")[0], pool.rows(0, "v")[0]
    at = (chosen.flatten().long()[:, None] * pool.size + torch.arange(pool.size, device=device)).flatten()
    at = at[at < int(pool.lens[0])]
    k, v = k[at], v[at]
    for part in range(0, 4096, 512):
        x = q[0, part:part + 512].double()
        want = torch.softmax((x @ k.t().contiguous()) * dim ** -0.5, -1) @ v
        size = (x.abs() @ k.abs().t().contiguous()).amax(-1, keepdim=True) * dim ** -0.5
        tol = want.abs() * 2.0 ** -11 + 2.0 ** -25 + float(v.abs().amax()) * (
            2 * (dim + 4) * 2.0 ** -24 * size + 2 * len(at) * 2.0 ** -24 + 2.0 ** -16)  # as in paged_reference.attention
        R.check(out[0, part:part + 512], want.cpu(), tol.cpu(), f"heads from {part}")
