"""Timed cases of the paged KV cache: rows written into pages and read back,
one new token attended over a sequence's pages, and the same over the pages
that a cheap score selects.

A case is a dict of plain sizes.  ``prepare`` makes what a serving program
holds before the call: the page pool, the block table, lengths and the new
rows or queries.  ``run`` is one pass:

* ``append``: new K/V rows of every sequence into its pages (8-bit pages:
  quantised with one scale per row, then read back, so that the outputs are the
  values the codes stand for), with each page's key bounds;
* ``read``: a range of positions of every sequence back into fp16 rows;
* ``attend``: one query token per sequence over all of its tokens;
* ``sparse``: pages chosen per KV head by the bound of q . k over the page,
  then the same attention over the chosen pages alone.

Definitions (P pages of S tokens, H KV heads, D coordinates, G query heads per
KV head; position p of sequence b is row p % S of page ``table[b, p // S]``):

* int8 page row: ``scale = amax / 127``, ``code = rint(x * (127 / amax))``;
  e4m3 the same with 448 and the format's own rounding; amax 0 gives zeros;
* bounds: per page, KV head and coordinate the smallest and largest key;
* page score: ``max over the group's heads of sum_d max(q_d, 0) * hi_d +
  min(q_d, 0) * lo_d``, rounded to 32 bits; ties go to the lowest page; the
  first and last pages are always kept; pages in ascending order, then -1;
* attention: ``softmax(scale * q . k) v`` over the allowed positions, zeros
  where there are none.
"""

from __future__ import annotations

import math
import random

import torch

own = False

MAXIMA = {"int8": 127.0, "e4m3": 448.0}
TYPES = {"fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # one decode step's K/V of 32 sequences (8 KV heads, D 64: the batched_32x32k shape), the latency of a small call
        {"name": "append_step_32", "op": "append", "type": "fp16", "batch": 32, "tokens": 1, "context": 2047,
         "ragged": False, "kv_heads": 8, "head_dim": 64, "page": 16, "pad": 0},
        # a prompt of the llama1b_8k shape into int8 pages, a ragged length, and its window read back
        {"name": "append_prompt_8k", "op": "append", "type": "int8", "batch": 1, "tokens": 8191, "context": 0,
         "ragged": False, "kv_heads": 8, "head_dim": 64, "page": 64, "pad": 0},
        # chunks of several prompts behind what they hold already, at the default configuration's 32 heads of 128;
        # the batch's rows are padded to a common size
        {"name": "append_ragged_e4m3", "op": "append", "type": "e4m3", "batch": 16, "tokens": 1000, "context": 777,
         "ragged": True, "kv_heads": 32, "head_dim": 128, "page": 32, "pad": 61},
        # the window of one sequence read back for a chunk of its prompt
        {"name": "read_32k", "op": "read", "type": "fp16", "batch": 1, "tokens": 32767, "ragged": False,
         "kv_heads": 8, "head_dim": 64, "page": 16},
        # windows of a ragged batch read back from 8-bit pages
        {"name": "read_ragged_int8", "op": "read", "type": "int8", "batch": 24, "tokens": 2500, "ragged": True,
         "kv_heads": 8, "head_dim": 128, "page": 32},
        # the smallest decode step: 8 heads, about 1,000 tokens (the smoke_1k shape)
        {"name": "attend_1k", "op": "attend", "type": "fp16", "batch": 1, "tokens": 1021, "ragged": False,
         "q_heads": 8, "kv_heads": 8, "head_dim": 64, "page": 16},
        # one sequence at the llama1b_8k shape, 8-bit pages
        {"name": "attend_8k_int8", "op": "attend", "type": "int8", "batch": 1, "tokens": 8192, "ragged": False,
         "q_heads": 32, "kv_heads": 8, "head_dim": 64, "page": 16},
        # batched serving, 32 sequences of 32,768 tokens
        {"name": "attend_32x32k", "op": "attend", "type": "fp16", "batch": 32, "tokens": 32768, "ragged": False,
         "q_heads": 32, "kv_heads": 8, "head_dim": 64, "page": 16},
        # a batch of very different lengths with 8 query heads per KV head (longctx_128k's heads)
        {"name": "attend_ragged_e4m3", "op": "attend", "type": "e4m3", "batch": 48, "tokens": 16000, "ragged": True,
         "q_heads": 32, "kv_heads": 4, "head_dim": 64, "page": 64},
        # the default configuration: 32 heads of 128, one query head per KV head
        {"name": "attend_mha_4x8k", "op": "attend", "type": "fp16", "batch": 4, "tokens": 8001, "ragged": False,
         "q_heads": 32, "kv_heads": 32, "head_dim": 128, "page": 32},
        # long context: 64 of 2,048 pages of one sequence of 131,072 tokens
        {"name": "sparse_128k_int8", "op": "sparse", "type": "int8", "batch": 1, "tokens": 131072, "ragged": False,
         "q_heads": 32, "kv_heads": 4, "head_dim": 64, "page": 64, "count": 64},
        # batched serving with 128 of up to 2,048 pages each
        {"name": "sparse_32x32k", "op": "sparse", "type": "fp16", "batch": 32, "tokens": 32768, "ragged": True,
         "q_heads": 32, "kv_heads": 8, "head_dim": 64, "page": 16, "count": 128},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "attend", "attend", "attend", "attend", "sparse", "sparse"])
    head_dim = rng.choice([64, 64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 32])
    batch = _log(rng, 1, 64)
    c = {"op": op, "type": rng.choice(["fp16", "fp16", "int8", "e4m3"]), "batch": batch,
         "ragged": rng.random() < 0.5, "kv_heads": kv_heads, "head_dim": head_dim,
         "page": rng.choice([16, 16, 32, 64, 128])}
    row = kv_heads * head_dim
    if op == "append":
        c["tokens"] = 1 if rng.random() < 0.3 else _log(rng, 2, min(16384, max(2, (16 << 20) // (batch * row))))
        c["context"] = 0 if rng.random() < 0.3 else _log(rng, 1, max(2, min(2048, (16 << 20) // (batch * row))))
        c["pad"] = rng.choice([0, 0, rng.randrange(1, 200)])
    elif op == "read":
        c["tokens"] = _log(rng, 1, min(32768, max(2, (64 << 20) // (batch * row))))
    else:
        c["q_heads"] = kv_heads * rng.choice([1, 2, 3, 4, 4, 8, 16])
        most = min(131072, max(2, (256 << 20) // (batch * row)))
        c["tokens"] = _log(rng, 1, most)
        if op == "sparse":
            c["tokens"] = max(c["tokens"], min(most, 20 * c["page"]))
            c["count"] = _log(rng, 2, max(2, -(-c["tokens"] // c["page"]) // 2))
    return c


def _counts(case):
    """Tokens per sequence that the call appends, reads or attends: a property of the case, not of the seed."""
    n, batch = case["tokens"], case["batch"]
    if not case["ragged"]:
        return [n] * batch
    rng = random.Random(1009 * batch + n)
    return [n if i == batch // 2 else _log(rng, 1, n) for i in range(batch)]


def _starts(case):
    """Tokens that a sequence holds before the call."""
    if case["op"] != "append":
        return [0] * case["batch"]
    rng = random.Random(77 * case["batch"] + case["context"])
    return [case["context"] if not case["ragged"] else rng.randint(0, case["context"]) for _ in range(case["batch"])]


def _rows(case, shape, g):
    """Rows of N(0, 1) with one scale per channel, U(0.5, 2), as the decode workloads draw keys and values."""
    scale = torch.rand((case["kv_heads"], case["head_dim"]), generator=g, device="cuda") * 1.5 + 0.5
    if len(shape) == 4:  # pages [P, H, S, D]
        scale = scale[:, None]
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) * scale.half()


def _quantise(x, kind):
    """Rows [..., D] fp16 -> (codes, scale [...] fp32)."""
    xf = x.float()
    amax = xf.abs().amax(-1)
    top = torch.full_like(amax, MAXIMA[kind])  # a tensor: torch divides by a number through its reciprocal
    inv = torch.where(amax > 0, top / amax, 0.0)
    y = xf * inv[..., None]
    codes = y.round().to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)
    return codes, amax / top


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = random.Random(seed)
    batch, heads, dim, size = case["batch"], case["kv_heads"], case["head_dim"], case["page"]
    counts, starts = _counts(case), _starts(case)
    need = [-(-(a + n) // size) for a, n in zip(starts, counts)]
    total = sum(need) + 3
    order = list(range(total))
    h.shuffle(order)
    width = max(need) + 2
    table = torch.full((batch, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    shape = (total, heads, size, dim)
    k, v = _rows(case, shape, g), _rows(case, shape, g)
    if case["op"] == "sparse":  # neighbouring tokens are alike: a page's keys share a part of their direction
        k = k * 0.6 + _rows(case, (total, heads, 1, dim), g)
    s = {"scale": dim ** -0.5, "type": case["type"], "page": size, "heads": heads, "table": table.cuda(),
         "bounds": torch.stack([k.amin(2), k.amax(2)], 2).contiguous(), "op": case["op"],
         "k_scale": None, "v_scale": None, "count": case.get("count", 0), "rows": sum(counts), "longest": max(counts)}
    if case["type"] != "fp16":
        k, s["k_scale"] = _quantise(k, case["type"])
        v, s["v_scale"] = _quantise(v, case["type"])
    s["k"], s["v"] = k, v
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    s["cu"] = torch.tensor(cu, dtype=torch.int32).cuda()
    if case["op"] == "append":
        s["lens"] = torch.tensor(starts, dtype=torch.int32).cuda()
        s["one"] = case["tokens"] == 1 and not case["pad"]
        new = (s["rows"] + case["pad"], heads, dim)
        s["k_new"], s["v_new"] = _rows(case, new, g), _rows(case, new, g)
    elif case["op"] == "read":
        s["lens"] = torch.tensor(starts, dtype=torch.int32).cuda()
    else:
        s["lens"] = torch.tensor(counts, dtype=torch.int32).cuda()
        s["q"] = torch.randn((batch, case["q_heads"], dim), generator=g, device="cuda", dtype=torch.float16)
    return s


def run(s):
    return _own(s) if own else PLAIN[s["op"]](s)


def _own(s):
    from apple_amd import kernels as K

    pages = K.KVPages(s["k"], s["v"], s["k_scale"], s["v_scale"], s["bounds"])
    if s["op"] == "append":
        K.paged_append(pages, s["table"], s["lens"], s["k_new"], s["v_new"], None if s["one"] else s["cu"])
        if s["type"] == "fp16":
            return {"k": s["k"], "v": s["v"], "bounds": s["bounds"]}
        k, v = K.paged_read(pages, s["table"], s["lens"], s["cu"], s["rows"])
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"], "bounds": s["bounds"]}
    if s["op"] == "read":
        k, v = K.paged_read(pages, s["table"], s["lens"], s["cu"], s["rows"])
        return {"k": k, "v": v}
    if s["op"] == "attend":
        return {"out": K.paged_attention(s["q"], pages, s["table"], s["lens"], s["scale"])}
    chosen = K.page_select(s["q"], pages, s["table"], s["lens"], s["count"], first=1, last=1)
    return {"chosen": chosen, "out": K.paged_attention(s["q"], pages, s["table"], s["lens"], s["scale"], chosen)}


# ------------------------------------------------------------------ plain form

def _places(s):
    """Page and row in the page of each of the call's rows."""
    n = torch.arange(s["rows"], device="cuda")
    cu = s["cu"].long()
    b = torch.searchsorted(cu[1:], n, right=True)
    pos = s["lens"].long()[b] + n - cu[b]
    return s["table"].long()[b, pos // s["page"]], pos % s["page"]


def _at(t, index):
    """t[index] in 32 bits."""
    return (t[index] if t.dtype != torch.float8_e4m3fn else t.view(torch.uint8)[index].view(t.dtype)).float()


def _window(s, index):
    """K and V rows [..., D] in 32 bits at an index of page, head and row."""
    k, v = _at(s["k"], index), _at(s["v"], index)
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][index][..., None], v * s["v_scale"][index][..., None]
    return k, v


def _plain_append(s):
    page, row = _places(s)
    k, v = s["k_new"][:s["rows"]], s["v_new"][:s["rows"]]
    first = page.new_zeros(len(s["k"]) + 1).bool()  # pages that begin with this call: their bounds are set, not widened
    first[torch.where(row == 0, page, len(s["k"]))] = True
    fresh = first[:-1, None, None]
    where = page[:, None, None].expand(k.shape)
    lo = torch.where(fresh, math.inf, s["bounds"][:, :, 0].float()).scatter_reduce(0, where, k.float(), "amin")
    hi = torch.where(fresh, -math.inf, s["bounds"][:, :, 1].float()).scatter_reduce(0, where, k.float(), "amax")
    s["bounds"].copy_(torch.stack([lo, hi], 2))
    if s["type"] == "fp16":
        s["k"][page, :, row] = k
        s["v"][page, :, row] = v
        return {"k": s["k"], "v": s["v"], "bounds": s["bounds"]}
    # codes are written as the bytes they are
    kc, ks = _quantise(k, s["type"])
    vc, vs = _quantise(v, s["type"])
    s["k"].view(torch.uint8)[page, :, row] = kc.view(torch.uint8)
    s["v"].view(torch.uint8)[page, :, row] = vc.view(torch.uint8)
    s["k_scale"][page, :, row] = ks
    s["v_scale"][page, :, row] = vs
    return _plain_read(s) | {"k_scale": s["k_scale"], "v_scale": s["v_scale"], "bounds": s["bounds"]}


def _plain_read(s):
    page, row = _places(s)
    k, v = _window(s, (page, slice(None), row))                            # [N, H, D]
    return {"k": k.half(), "v": v.half()}


def _softmax_v(q, k, v, allowed, scale):
    """q [B, H, G, D]; k, v [B, H, T, D]; allowed [B, 1 or H, T]."""
    score = torch.matmul(q, k.transpose(-1, -2)) * scale
    score = torch.where(allowed[:, :, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, torch.where(allowed[..., None], v, 0.0)) / total
    return torch.where(total == 0, 0.0, out)


def _heads(s):
    batch, q_heads, dim = s["q"].shape
    return s["q"].float().view(batch, s["heads"], q_heads // s["heads"], dim)


def _plain_attend(s):
    pos = torch.arange(s["longest"], device="cuda")
    page = s["table"].long()[:, pos // s["page"]].clamp_min(0)
    row = (pos % s["page"]).expand(page.shape)
    k, v = _window(s, (page, slice(None), row))                            # [B, T, H, D]
    allowed = (pos < s["lens"][:, None])[:, None]
    out = _softmax_v(_heads(s), k.transpose(1, 2), v.transpose(1, 2), allowed, s["scale"])
    return {"out": out.reshape(s["q"].shape).half()}


def _plain_select(s):
    """Chosen pages [B, H, count], in 64 bits: the score of a page may lie next to the last kept one's."""
    size, table = s["page"], s["table"].long()
    held = (s["lens"].long() + size - 1) // size                           # [B]
    near = s["bounds"][table.clamp_min(0)].double()                        # [B, W, H, 2, D]
    q = _heads(s).double().transpose(-1, -2)                               # [B, H, D, G]
    score = (torch.matmul(near[:, :, :, 1].transpose(1, 2), q.clamp_min(0))
             + torch.matmul(near[:, :, :, 0].transpose(1, 2), q.clamp_max(0))).amax(-1)  # [B, H, W]
    score = score.float().double().nan_to_num(1e300, 1e300, -1e300)
    n = torch.arange(table.shape[1], device="cuda")
    kept = (n < 1) | (n >= held[:, None] - 1)
    score = torch.where(kept[:, None], math.inf, score)
    score = torch.where((n < held[:, None])[:, None], score, -math.inf)
    order = torch.sort(-score, dim=-1, stable=True).indices[..., :s["count"]]
    order = torch.where(order < held[:, None, None], order, table.shape[1]).sort(-1).values
    order = torch.where(order < table.shape[1], order, -1)
    missing = s["count"] - order.shape[-1]
    return torch.nn.functional.pad(order, (0, max(0, missing)), value=-1)


def _plain_sparse(s):
    chosen = _plain_select(s)                                              # [B, H, count]
    batch, heads, count = chosen.shape
    b = torch.arange(batch, device="cuda")[:, None, None]
    h = torch.arange(heads, device="cuda")[None, :, None]
    page = s["table"].long()[b, chosen.clamp_min(0)].clamp_min(0)
    k, v = _window(s, (page, h))                                           # [B, H, count, S, D]
    pos = chosen[..., None] * s["page"] + torch.arange(s["page"], device="cuda")
    allowed = (chosen[..., None] >= 0) & (pos < s["lens"][:, None, None, None])
    flat = (batch, heads, count * s["page"])
    out = _softmax_v(_heads(s), k.reshape(*flat, -1), v.reshape(*flat, -1), allowed.reshape(flat), s["scale"])
    return {"chosen": chosen.int(), "out": out.reshape(s["q"].shape).half()}


PLAIN = {"append": _plain_append, "read": _plain_read, "attend": _plain_attend, "sparse": _plain_sparse}


# ------------------------------------------------------------------ work and exact results

def work(case):
    counts = _counts(case)
    heads, dim = case["kv_heads"], case["head_dim"]
    wide = 2 if case["type"] == "fp16" else 1
    stored = heads * (dim * wide + (0 if wide == 2 else 4)) * 2            # K and V of one token, scales with them
    plain = heads * dim * 2 * 2                                            # the same as fp16 rows
    n = sum(counts)
    if case["op"] == "append":
        runs = sum(-(-(a + m) // case["page"]) - a // case["page"] for a, m in zip(_starts(case), counts))
        moved = n * (plain + stored) + runs * heads * dim * 2 * 2
        if wide == 1:  # and read back
            moved += n * (plain + stored)
        return {"bytes": moved, "flops": 4 * n * heads * dim}
    if case["op"] == "read":
        return {"bytes": n * (plain + stored), "flops": 2 * n * heads * dim}
    q_heads = case["q_heads"]
    ends = case["batch"] * q_heads * dim * 2 * 2
    if case["op"] == "attend":
        return {"bytes": n * stored + ends, "flops": 4 * n * q_heads * dim}
    pages = sum(-(-m // case["page"]) for m in counts)
    seen = sum(min(m, case["count"] * case["page"]) for m in counts)
    return {"bytes": pages * heads * dim * 2 * 2 + seen * stored + ends,
            "flops": 4 * pages * q_heads * dim + 4 * seen * q_heads * dim}


def exact(case, seed):
    """Results in 64 bits, a sequence at a time."""
    s = prepare(case, seed)
    counts, starts = _counts(case), _starts(case)
    size, heads, dim = case["page"], case["kv_heads"], case["head_dim"]

    def stored(codes, scale):
        x = codes.to(torch.float32).double()
        return x if scale is None else x * scale.double()[..., None]

    def window(b, begin, end):
        """K and V [H, end - begin, D] of sequence b."""
        ids = s["table"][b, begin // size:-(-end // size)].long()
        off = begin - begin // size * size
        pick = []
        for name in ("k", "v"):
            codes = s[name].view(torch.uint8)[ids].view(s[name].dtype) if case["type"] == "e4m3" else s[name][ids]
            x = stored(codes, None if s[name + "_scale"] is None else s[name + "_scale"][ids])
            pick.append(x.transpose(0, 1).reshape(heads, -1, dim)[:, off:off + end - begin])
        return pick

    def attend(q, k, v):
        """q [H, G, D]; k, v [H, T, D]."""
        if k.shape[1] == 0:
            return torch.zeros_like(q)
        score = torch.bmm(q, k.transpose(1, 2).contiguous()) * s["scale"]
        return torch.bmm(torch.softmax(score, -1), v)

    if case["op"] in ("append", "read"):
        parts = []
        if case["op"] == "append":
            lo, hi = s["bounds"][:, :, 0].double(), s["bounds"][:, :, 1].double()
            pools, scales, at = {}, {}, 0
            for name in ("k", "v"):
                pools[name] = stored(s[name], None) if case["type"] == "fp16" else None
                scales[name] = None if s[name + "_scale"] is None else s[name + "_scale"].double()
            for b, (a, m) in enumerate(zip(starts, counts)):
                new = {name: s[name + "_new"][at:at + m].double() for name in ("k", "v")}
                at += m
                read = {}
                for name, x in new.items():
                    read[name] = x
                    if case["type"] != "fp16":
                        top = MAXIMA[case["type"]]
                        step = x.abs().amax(-1, keepdim=True) / top
                        y = torch.where(step > 0, x / step, 0.0)
                        if case["type"] == "int8":
                            y = y.round()
                        else:  # three bits behind the leading one, from 2^-6 up
                            unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
                            y = (y / unit).round() * unit
                        read[name] = y * step
                for p in range(a // size, -(-(a + m) // size)):
                    i0, i1 = max(0, p * size - a), min(m, (p + 1) * size - a)
                    page, r0 = int(s["table"][b, p]), max(0, a - p * size)
                    low, high = new["k"][i0:i1].amin(0), new["k"][i0:i1].amax(0)
                    lo[page] = low if r0 == 0 else torch.minimum(lo[page], low)
                    hi[page] = high if r0 == 0 else torch.maximum(hi[page], high)
                    for name, x in new.items():
                        if case["type"] == "fp16":
                            pools[name][page, :, r0:r0 + i1 - i0] = x[i0:i1].transpose(0, 1)
                        else:
                            scales[name][page, :, r0:r0 + i1 - i0] = (x[i0:i1].abs().amax(-1) / top).transpose(0, 1)
                parts.append(read)
            bounds = torch.stack([lo, hi], 2)
            if case["type"] == "fp16":
                return {"k": pools["k"], "v": pools["v"], "bounds": bounds}
            return {"k": torch.cat([p["k"] for p in parts]), "v": torch.cat([p["v"] for p in parts]),
                    "k_scale": scales["k"], "v_scale": scales["v"], "bounds": bounds}
        for b, m in enumerate(counts):
            k, v = window(b, 0, m)
            parts.append((k.transpose(0, 1), v.transpose(0, 1)))
        return {"k": torch.cat([p[0] for p in parts]), "v": torch.cat([p[1] for p in parts])}

    outs, picked = [], []
    for b, m in enumerate(counts):
        q = s["q"][b].double().view(heads, -1, dim)
        k, v = window(b, 0, m)
        if case["op"] == "sparse":
            n = -(-m // size)
            low, high = (s["bounds"][s["table"][b, :n].long()].double().transpose(0, 1)[:, :, i] for i in (0, 1))
            score = torch.zeros((heads, n, q.shape[1]), dtype=torch.float64, device="cuda")
            for i in range(dim):
                qi = q[:, None, :, i]
                score += torch.where(qi >= 0, qi * high[:, :, None, i], qi * low[:, :, None, i])
            score = score.amax(-1)
            score[:, 0] = score[:, -1] = math.inf
            keep = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :case["count"]].sort(-1).values
            picked.append(torch.nn.functional.pad(keep, (0, case["count"] - keep.shape[1]), value=-1).int())
            tokens = torch.zeros((heads, n), dtype=torch.bool, device="cuda").scatter_(1, keep, True)
            tokens = tokens.repeat_interleave(size, 1)[:, :m]
            outs.append(torch.cat([attend(q[h:h + 1], k[h:h + 1, tokens[h]], v[h:h + 1, tokens[h]])
                                   for h in range(heads)]).reshape(-1, dim))
        else:
            outs.append(attend(q, k, v).reshape(-1, dim))
    out = torch.stack(outs)
    return {"chosen": torch.stack(picked), "out": out} if case["op"] == "sparse" else {"out": out}
