"""The paged KV cache's operators restated in 64 bits on the host, one sequence,
head and page at a time."""

import math

import numpy as np
import torch

MAXIMA = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
KINDS = {"fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def quantise(x, dtype):
    """Rows [..., D] fp16 -> (codes, scales fp32): one fp32 division for the
    scale, one for its reciprocal, one product per value; a row with a value
    that is not finite has scale NaN and codes 0."""
    xf = x.float()
    amax = xf.abs().amax(-1)
    top = torch.full_like(amax, MAXIMA[dtype])  # a tensor: torch divides by a number through its reciprocal
    fine = torch.isfinite(xf).all(-1)
    inv = torch.where(fine & (amax > 0), top / amax, torch.zeros_like(amax))
    y = torch.where(fine[..., None], xf * inv[..., None], torch.zeros_like(xf))
    codes = y.round().to(torch.int8) if dtype == torch.int8 else y.to(torch.float8_e4m3fn)
    return codes, torch.where(fine, amax / top, torch.full_like(amax, math.nan))


class Pool:
    """A page pool on the host; ``pages()`` is the same on a device."""

    def __init__(self, kind, pages, heads, size, dim, seed, bounds=True):
        self.g = torch.Generator().manual_seed(seed)
        self.kind, self.size, self.heads, self.dim, self.count = kind, size, heads, dim, pages
        shape = (pages, heads, size, dim)
        k, v = self.randn(shape), self.randn(shape)
        self.bounds = torch.stack([k.amin(2), k.amax(2)], 2).contiguous() if bounds else None
        self.k_scale = self.v_scale = None
        if kind != "fp16":
            k, self.k_scale = quantise(k, KINDS[kind])
            v, self.v_scale = quantise(v, KINDS[kind])
        self.k, self.v = k, v

    def randn(self, shape, scale=1.0):
        return (torch.randn(shape, generator=self.g) * scale).half()

    def tables(self, lens, spare=2):
        """A table of distinct pages in a shuffled order, -1 behind each sequence's last."""
        need = [-(-n // self.size) for n in lens]
        order = torch.randperm(self.count, generator=self.g).tolist()
        assert sum(need) <= self.count
        table = torch.full((len(lens), max(need, default=0) + spare), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        return table

    def pages(self, device):
        from apple_amd.kernels import KVPages

        return KVPages(*(None if t is None else t.to(device)
                         for t in (self.k, self.v, self.k_scale, self.v_scale, self.bounds)))

    def values(self, name):
        """[P, H, S, D] in 64 bits."""
        x = getattr(self, name).float().double()
        s = getattr(self, name + "_scale")
        return x if s is None else x * s.double()[..., None]

    def append(self, table, lens, k, v, cu):
        width = table.shape[1]
        for b in range(len(lens)):
            for i in range(cu[b], min(cu[b + 1], len(k))):
                pos = lens[b] + i - cu[b]
                page = int(table[b, pos // self.size]) if pos // self.size < width else -1
                if not 0 <= page < self.count:
                    continue
                row = pos % self.size
                for name, x in (("k", k[i]), ("v", v[i])):
                    t = getattr(self, name)
                    if self.kind == "fp16":
                        t[page, :, row] = x
                    else:
                        codes, scale = quantise(x, KINDS[self.kind])
                        t.view(torch.uint8)[page, :, row] = codes.view(torch.uint8)
                        getattr(self, name + "_scale")[page, :, row] = scale
                if self.bounds is not None:
                    lo, hi = self.bounds[page, :, 0], self.bounds[page, :, 1]
                    new = k[i]
                    self.bounds[page, :, 0] = new if row == 0 else torch.minimum(lo, new)
                    self.bounds[page, :, 1] = new if row == 0 else torch.maximum(hi, new)

    def window(self, table, b, begin, end):
        """(values K, V [end - begin, H, D] in 64 bits, whether there is a page)."""
        out = [torch.zeros((end - begin, self.heads, self.dim), dtype=torch.float64) for _ in range(2)]
        there = torch.zeros(end - begin, dtype=torch.bool)
        kk, vv = self.values("k"), self.values("v")
        for i in range(end - begin):
            o = (begin + i) // self.size
            page = int(table[b, o]) if 0 <= o < table.shape[1] else -1
            if 0 <= page < self.count:
                there[i] = True
                out[0][i], out[1][i] = kk[page, :, (begin + i) % self.size], vv[page, :, (begin + i) % self.size]
        return out[0], out[1], there


def softmax_v(q, k, v, scale):
    """q [D], k, v [T, D] in 64 bits -> (out, the bound on sum |q k| scale)."""
    if len(k) == 0:
        return torch.zeros_like(q), 0.0
    s = (k * q).sum(-1) * scale
    top = s.amax()
    p = torch.exp(s - (top if top != -math.inf else 0.0))
    p = torch.where(p < 2.0 ** -149, 0.0, p)  # weights are fp32: what is under its smallest value is 0 (0 * inf: NaN)
    total = p.sum()
    out = (p[:, None] * v).sum(0) / total
    size = float(((k * q).abs().sum(-1) * abs(scale)).nan_to_num(0, 0, 0).max())
    return (torch.zeros_like(q) if total == 0 else out), size


def attention(pool, table, lens, q, scale, chosen=None):
    """(out [B, Hq, D] in 64 bits, tolerance of the same shape).

    The tolerance counts, per output: half a step of fp16 (2^-11 of the value,
    2^-25 below its normal range); a score's fp32 error of at most (D + 4) 2^-24
    of sum |q k| scale, which moves a weight by as much of itself and so the
    output by at most twice that times the largest |v|; sums of T weights, T 2^-24
    of the largest |v| for each of numerator and denominator; weights kept to
    2^-16 of themselves."""
    B, Hq, D = q.shape
    G = Hq // pool.heads
    out, tol = torch.zeros((B, Hq, D), dtype=torch.float64), torch.zeros((B, Hq, D), dtype=torch.float64)
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * pool.size))
        k, v, there = pool.window(table, b, 0, n)
        for i in range(Hq):
            h = i // G
            if chosen is None:
                at = torch.arange(n)
            else:
                at = torch.tensor([p * pool.size + r for p in chosen[b, h].tolist() if p >= 0
                                   for r in range(pool.size) if p * pool.size + r < n], dtype=torch.long)
            at = at[there[at]] if len(at) else at
            kk, vv = k[at, h], v[at, h]
            out[b, i], size = softmax_v(q[b, i].double(), kk, vv, scale)
            big = float(vv.abs().nan_to_num(0, 0, 0).max()) if len(at) else 0.0
            tol[b, i] = (out[b, i].abs().nan_to_num(0, 0, 0) * 2.0 ** -11 + 2.0 ** -25
                         + big * (2 * (D + 4) * 2.0 ** -24 * size + 2 * len(at) * 2.0 ** -24 + 2.0 ** -16))
    return out, tol


def check(got, want, tol, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    # past fp16's largest value a result rounds to infinity
    far = want.abs() > 65519.0
    want = torch.where(far & torch.isfinite(want), torch.sign(want) * math.inf, want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fine = torch.isfinite(want)
    rest = ~fine & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest]), what
    off = (got - want).abs()[fine] - tol[fine]
    assert not off.numel() or float(off.max()) <= 0.0, (what, float((got - want).abs()[fine].max()), float(off.max()))


def select(pool, table, lens, q, count, first, last):
    """Chosen pages [B, Hkv, count]: scores in 64 bits, rounded to 32."""
    B, Hq, D = q.shape
    G = Hq // pool.heads
    out = np.full((B, pool.heads, count), -1, dtype=np.int32)
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * pool.size))
        held = -(-n // pool.size)
        for h in range(pool.heads):
            score = []
            for o in range(held):
                page = int(table[b, o])
                if not 0 <= page < pool.count:
                    score.append(-math.inf)
                    continue
                lo, hi = pool.bounds[page, h].double()
                x = q[b, h * G:(h + 1) * G].double()
                up, down = torch.where(x < 0, 0.0, x), torch.where(x > 0, 0.0, x)
                s = float((up * hi + down * lo).sum(-1).amax().float())
                score.append(math.inf if math.isnan(s) else s)
            kept = [o for o in range(held) if o < first or o >= held - last]
            rest = sorted((o for o in range(held) if o not in set(kept)), key=lambda o: (-score[o], o))
            pick = sorted((kept + rest)[:count])
            out[b, h, :len(pick)] = pick
    return torch.from_numpy(out)
