"""What bounds a paged cache's memory, restated in 64 bits on the host: pages of
4-bit floats, accumulated attention weights, eviction by them, and rotary
positions."""

import math

import torch

from tests import paged_reference as R

MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
SCALES = (torch.arange(256, dtype=torch.int16) << 7).view(torch.float16).double()  # by byte; 249 .. 255 are NaN
TOP = 0xE2                                                                          # the byte of 10240, the largest scale
KINDS = ("fp16", "int8", "e4m3", "e2m1")


def nearest(x, table):
    """Index of the nearest entry of an ascending table, ties to the even index."""
    off = (x[..., None] - table).abs()
    best = off.amin(-1, keepdim=True)
    index = torch.arange(len(table)).expand(off.shape)
    first = torch.where(off == best, index, len(table)).amin(-1)
    after = torch.where(off == best, index, -1).amax(-1)
    return torch.where(first % 2 == 0, first, after)


def quantise4(x):
    """Rows [..., D] fp16 -> (codes, two a byte [..., D / 2], scale bytes [..., D / 16])."""
    g = x.double().unflatten(-1, (-1, 16))
    fine = torch.isfinite(g).all(-1)
    amax = torch.where(fine, g.abs().nan_to_num(0, 0, 0).amax(-1), 0.0)
    byte = nearest(amax / 6, SCALES[:TOP + 1])
    scale = SCALES[byte][..., None]
    fine = fine[..., None]
    live = fine & (scale > 0)
    a = torch.where(live, g.abs().nan_to_num(0, 0, 0) / scale, 0.0)
    code = nearest(a.clamp_max(6.0), MAGNITUDES) | torch.where(torch.signbit(g) & live, 8, 0)
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return (code[..., 0] | code[..., 1] << 4).to(torch.uint8), torch.where(fine[..., 0], byte, 255).to(torch.uint8)


def values4(codes, scales):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = torch.where(c > 7, -MAGNITUDES[c % 8], MAGNITUDES[c % 8])
    return (v.unflatten(-1, (-1, 16)) * SCALES[scales.long()][..., None]).flatten(-2)


class Pool(R.Pool):
    """A page pool of any type with accumulated weights."""

    def __init__(self, kind, pages, heads, size, dim, seed, bounds=True):
        super().__init__("fp16" if kind == "e2m1" else kind, pages, heads, size, dim, seed, bounds)
        if kind == "e2m1":
            self.kind = kind
            self.k, self.k_scale = quantise4(self.k)
            self.v, self.v_scale = quantise4(self.v)
        # few rows with most of the weight, some without any, some alike
        w = torch.exp(2.0 * torch.randn((pages, heads, size), generator=self.g))
        w = torch.where(torch.rand(w.shape, generator=self.g) < 0.1, 0.0, w)
        self.weight = torch.where(torch.rand(w.shape, generator=self.g) < 0.2, 0.25, w)

    def values(self, name):
        if self.kind != "e2m1":
            return super().values(name)
        return values4(getattr(self, name), getattr(self, name + "_scale"))

    def tensors(self):
        return {n: getattr(self, n) for n in ("k", "v", "k_scale", "v_scale", "bounds", "weight") if getattr(self, n) is not None}

    def poison(self, table, lens):
        """NaN in every row that no sequence holds."""
        held = torch.zeros((self.count, self.size), dtype=torch.bool)
        for b, n in enumerate(lens):
            for i in range(min(max(n, 0), table.shape[1] * self.size)):
                page = int(table[b, i // self.size])
                if 0 <= page < self.count:
                    held[page, i % self.size] = True
        free = (~held)[:, None, :].expand(-1, self.heads, -1)
        self.weight[free] = math.nan
        for name in ("k", "v"):
            if self.kind == "fp16":
                getattr(self, name)[free] = math.nan
            elif self.kind == "e2m1":
                getattr(self, name + "_scale")[free] = 255
            else:
                getattr(self, name + "_scale")[free] = math.nan
        return self

    def append(self, table, lens, k, v, cu):
        if self.kind != "e2m1":
            super().append(table, lens, k, v, cu)
        for b in range(len(lens)):
            for i in range(cu[b], min(cu[b + 1], len(k))):
                pos = lens[b] + i - cu[b]
                page = int(table[b, pos // self.size]) if pos // self.size < table.shape[1] else -1
                if not 0 <= page < self.count:
                    continue
                row = pos % self.size
                self.weight[page, :, row] = 0
                if self.kind != "e2m1":
                    continue
                self.k[page, :, row], self.k_scale[page, :, row] = quantise4(k[i])
                self.v[page, :, row], self.v_scale[page, :, row] = quantise4(v[i])
                if self.bounds is not None:
                    lo, hi = self.bounds[page, :, 0], self.bounds[page, :, 1]
                    self.bounds[page, :, 0] = k[i] if row == 0 else torch.minimum(lo, k[i])
                    self.bounds[page, :, 1] = k[i] if row == 0 else torch.maximum(hi, k[i])

    def weigh(self, table, lens, q, scale):
        """Adds every position's softmax weights; returns the tolerance of the sums.

        A weight e^(s - m) / l: the score's fp32 error of at most (D + 4) 2^-24 of sum |q k| scale on either side of the
        difference, the sum's T 2^-24, an exponential and a quotient of a few steps each; adding G of them and what
        was there before, half a step of the sum each."""
        G = q.shape[1] // self.heads
        tol = torch.zeros(self.weight.shape, dtype=torch.float64)
        total = self.weight.double()
        for b in range(q.shape[0]):
            n = max(0, min(int(lens[b]), table.shape[1] * self.size))
            k, _, there = self.window(table, b, 0, n)
            at = torch.nonzero(there).flatten()
            if not len(at):
                continue
            page, row = table[b].long()[at // self.size], at % self.size
            for i in range(q.shape[1]):
                x = k[at, i // G] * q[b, i].double()
                s = x.sum(-1) * scale
                top = s.amax()
                if top == -math.inf:
                    continue
                p = torch.exp(s - top)
                w = p / p.sum()
                size = float((x.abs().sum(-1) * abs(scale)).nan_to_num(0, 0, 0).max())
                total[page, i // G, row] += w
                tol[page, i // G, row] += w.nan_to_num(0) * (2 * (self.dim + 4) * size + len(at) + 16) * 2.0 ** -24 + 2.0 ** -126
        tol += total.abs().nan_to_num(0) * (G + 1) * 2.0 ** -24
        self.weight = total
        return tol

    def evict(self, table, lens, keep, first, last):
        """The pool after an eviction; returns the new lengths."""
        new = []
        rows = {n: t for n, t in self.tensors().items() if n != "bounds"}
        for b, n in enumerate(lens):
            n = max(0, min(int(n), table.shape[1] * self.size))
            new.append(min(n, keep))
            if n <= keep:
                continue
            place = []
            for t in range(n):
                page = int(table[b, t // self.size])
                place.append((page, t % self.size) if 0 <= page < self.count else None)
            for h in range(self.heads):
                w = [-math.inf if p is None else float(self.weight[p[0], h, p[1]]) for p in place]
                w = [math.inf if math.isnan(x) else x for x in w]
                middle = sorted(range(first, n - last), key=lambda t: (-w[t], t))[:keep - first - last]
                kept = list(range(first)) + sorted(middle) + list(range(n - last, n))
                old = {name: [None if place[t] is None else t_[place[t][0], h, place[t][1]].clone() for t in kept]
                       for name, t_ in rows.items()}
                for j, t in enumerate(kept):
                    if place[j] is None:
                        continue
                    for name, t_ in rows.items():
                        x = old[name][j]
                        t_[place[j][0], h, place[j][1]] = torch.zeros_like(t_[0, 0, 0]) if x is None else x
            if self.bounds is not None:
                keys = self.values("k").half()
                for o in range(-(-keep // self.size)):
                    page = int(table[b, o])
                    if 0 <= page < self.count:
                        x = keys[page, :, :min(self.size, keep - o * self.size)]
                        self.bounds[page] = torch.stack([x.amin(1), x.amax(1)], 1)
        return new


def rotary(x, positions, inv_freq, layout, factor):
    """x [N, H, D] -> the same in 64 bits."""
    y = x.double().clone()
    r = 2 * len(inv_freq)
    angle = (positions.double()[:, None] * inv_freq)[:, None]
    a, b = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    c, s = torch.cos(angle) * factor, torch.sin(angle) * factor
    y[..., a], y[..., b] = x[..., a].double() * c - x[..., b].double() * s, x[..., b].double() * c + x[..., a].double() * s
    return y
