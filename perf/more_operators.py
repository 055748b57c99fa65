"""Timed cases of a paged KV cache in bounded memory: rotary positions of new
rows, pages of 4-bit floats, attention that adds up the weight of every position,
and eviction by that weight.

A case is a dict of plain sizes.  ``prepare`` makes what a serving program
holds before the call; ``run`` is one pass:

* ``rotary``: queries and keys of new rows at positions of their own;
* ``append``: new K/V rows of every sequence into 4-bit pages, and back into
  fp16 rows, so that the outputs are the values the codes stand for;
* ``attend``: one query per sequence over all of its tokens in 4-bit pages;
* ``weigh``: the same over pages of any type, each position's softmax weights
  added to its accumulated weight;
* ``evict``: sequences longer than ``keep`` give up, per KV head, the positions
  of the smallest accumulated weight.

Definitions (P pages of S tokens, H KV heads, D coordinates; position p of
sequence b is row p % S of page ``table[b, p // S]``):

* rotary: the first R coordinates in pairs (i, i + R/2) ("half") or (2i, 2i + 1)
  ("interleaved"): (x1, x2) -> factor (x1 cos a - x2 sin a, x2 cos a + x1 sin a),
  a = position * inv_freq[i];
* e2m1 row: per 16 coordinates a scale of 3 mantissa bits and fp16's exponents,
  ``scale = min(rn(amax / 6), 10240)``, kept as the byte ``fp16 bits >> 7``, and
  codes ``rn(x / scale)`` to sign and 0, .5, 1, 1.5, 2, 3, 4 or 6, ties to the
  even code, two a byte with the earlier coordinate in the low half;
* int8 / e4m3 row: ``scale = amax / 127`` (448), ``code = rn(x * (127 / amax))``;
* attention: ``softmax(scale * q . k) v``, zeros without positions; a position's
  weight grows by its softmax weights over the KV head's query heads;
* eviction: kept are the ``first`` oldest and ``last`` newest positions and the
  heaviest others, ties to the older, ``keep`` in all; they move to positions 0,
  1, ... in their order, rows behind stay as they are.
"""

from __future__ import annotations

import math
import random

import torch

own = False

MAXIMA = {"int8": 127.0, "e4m3": 448.0}
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # one new token of one sequence at the end of a long context (32 / 4 heads of 64: longctx_128k), latency
        {"name": "rotary_step_1", "op": "rotary", "type": "fp16", "batch": 1, "tokens": 1, "context": 131071,
         "q_heads": 32, "kv_heads": 4, "head_dim": 64, "rotary_dim": 64, "layout": "half", "stretch": 32.0, "factor": 1.0},
        # a prompt of the llama1b_8k shape, an odd length
        {"name": "rotary_prompt_8k", "op": "rotary", "type": "fp16", "batch": 1, "tokens": 8191, "context": 0,
         "q_heads": 32, "kv_heads": 8, "head_dim": 64, "rotary_dim": 64, "layout": "half", "stretch": 1.0, "factor": 1.0},
        # chunks of 16 prompts behind what they hold, the default configuration's heads, half of each rotated in pairs of
        # neighbours, positions stretched by 4 with the factor that goes with it
        {"name": "rotary_ragged_16k", "op": "rotary", "type": "bf16", "batch": 16, "tokens": 16384, "context": 30000,
         "q_heads": 32, "kv_heads": 32, "head_dim": 128, "rotary_dim": 64, "layout": "interleaved", "stretch": 4.0,
         "factor": 1.1386},
        # one decode step's rows of 32 sequences (batched_32x32k's heads), latency
        {"name": "e2m1_append_32", "op": "append", "type": "e2m1", "batch": 32, "tokens": 1, "context": 2047,
         "ragged": False, "kv_heads": 8, "head_dim": 64, "page": 16, "pad": 0},
        # chunks of several prompts at the default configuration's 32 heads of 128, the batch padded
        {"name": "e2m1_append_ragged", "op": "append", "type": "e2m1", "batch": 16, "tokens": 1000, "context": 777,
         "ragged": True, "kv_heads": 32, "head_dim": 128, "page": 32, "pad": 61},
        # one sequence at the llama1b_8k shape
        {"name": "e2m1_attend_8k", "op": "attend", "type": "e2m1", "batch": 1, "tokens": 8192, "ragged": False,
         "q_heads": 32, "kv_heads": 8, "head_dim": 64, "page": 16},
        # batched serving, 32 sequences of 32,768 tokens
        {"name": "e2m1_attend_32x32k", "op": "attend", "type": "e2m1", "batch": 32, "tokens": 32768, "ragged": False,
         "q_heads": 32, "kv_heads": 8, "head_dim": 64, "page": 16},
        # a batch of very different lengths at the default configuration's heads
        {"name": "e2m1_attend_ragged", "op": "attend", "type": "e2m1", "batch": 24, "tokens": 12001, "ragged": True,
         "q_heads": 32, "kv_heads": 32, "head_dim": 128, "page": 64},
        # one decode step that keeps count of the weights, one sequence
        {"name": "weigh_8k", "op": "weigh", "type": "e2m1", "batch": 1, "tokens": 8191, "ragged": False,
         "q_heads": 32, "kv_heads": 8, "head_dim": 64, "page": 16},
        # the same for a ragged batch, with 8 query heads per KV head
        {"name": "weigh_ragged_fp16", "op": "weigh", "type": "fp16", "batch": 32, "tokens": 20000, "ragged": True,
         "q_heads": 32, "kv_heads": 4, "head_dim": 64, "page": 64},
        # one sequence that has passed its budget by a page
        {"name": "evict_2k", "op": "evict", "type": "fp16", "batch": 1, "tokens": 2111, "ragged": False,
         "kv_heads": 8, "head_dim": 64, "page": 64, "keep": 2048, "first": 4, "last": 256},
        # prompts of a batch cut to 4,096 tokens each, the shorter ones left alone
        {"name": "evict_ragged_e2m1", "op": "evict", "type": "e2m1", "batch": 32, "tokens": 16000, "ragged": True,
         "kv_heads": 8, "head_dim": 128, "page": 32, "keep": 4096, "first": 4, "last": 512},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "append", "attend", "attend", "attend", "weigh", "weigh", "evict", "evict"])
    head_dim = rng.choice([64, 64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 32])
    batch = _log(rng, 1, 64)
    row = kv_heads * head_dim
    if op == "rotary":
        group = rng.choice([1, 2, 3, 4, 8])
        most = max(2, (64 << 20) // (row * (group + 1)))
        tokens = _log(rng, 1, min(16384, most))
        return {"op": op, "type": rng.choice(["fp16", "fp16", "bf16", "fp32"]), "batch": min(batch, tokens),
                "tokens": tokens, "context": rng.choice([0, 8191, _log(rng, 1, 1 << 20)]), "q_heads": kv_heads * group,
                "kv_heads": kv_heads, "head_dim": head_dim,
                "rotary_dim": rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4, 2 * rng.randrange(1, head_dim // 2)]),
                "layout": rng.choice(["half", "interleaved"]), "stretch": rng.choice([1.0, 4.0, 32.0]),
                "factor": rng.choice([1.0, 1.0, 1.1386])}
    c = {"op": op, "type": "e2m1", "batch": batch, "ragged": rng.random() < 0.5, "kv_heads": kv_heads,
         "head_dim": head_dim, "page": rng.choice([16, 16, 32, 64, 128])}
    if op == "append":
        c["tokens"] = 1 if rng.random() < 0.3 else _log(rng, 2, min(16384, max(2, (16 << 20) // (batch * row))))
        c["context"] = 0 if rng.random() < 0.3 else _log(rng, 1, max(2, min(2048, (16 << 20) // (batch * row))))
        c["pad"] = rng.choice([0, 0, rng.randrange(1, 200)])
        return c
    if op in ("weigh", "evict"):
        c["type"] = rng.choice(["fp16", "fp16", "int8", "e4m3", "e2m1", "e2m1"])
    if op == "evict":
        c["tokens"] = _log(rng, 2, min(32768, max(2, (64 << 20) // (batch * row))))
        c["keep"] = max(1, int(c["tokens"] * rng.choice([rng.uniform(0.05, 1.0), 0.5, 0.97])))
        c["first"] = min(rng.choice([0, 1, 4]), c["keep"])
        c["last"] = rng.randint(0, (c["keep"] - c["first"]) // 2)
        return c
    c["q_heads"] = kv_heads * rng.choice([1, 2, 3, 4, 4, 8, 16])
    c["tokens"] = _log(rng, 1, min(131072, max(2, ((256 if op == "attend" else 128) << 20) // (batch * row))))
    return c


def _counts(case):
    """Tokens per sequence that the call appends, attends or holds: a property of the case, not of the seed."""
    n, batch = case["tokens"], case["batch"]
    if not case["ragged"]:
        return [n] * batch
    rng = random.Random(1009 * batch + n)
    return [n if i == batch // 2 else _log(rng, 1, n) for i in range(batch)]


def _starts(case):
    """Tokens that a sequence holds before an append."""
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
    """Rows [..., D] fp16 -> (codes, scales): [..., D] and [...] fp32 of 8 bits, [..., D / 2] and [..., D / 16] bytes of 4."""
    xf = x.float()
    if kind == "e2m1":
        xf = xf.unflatten(-1, (-1, 16))
        amax = xf.abs().amax(-1)
        s = amax / torch.full_like(amax, 6.0)  # a tensor: torch divides by a number through its reciprocal
        unit = torch.exp2((torch.frexp(s).exponent - 1).clamp_min(-14).float() - 3.0)
        s = ((s / unit).round() * unit).clamp_max(10240.0)
        a = torch.where(s[..., None] > 0, xf.abs() / s[..., None], 0.0)
        # steps of 1/2 up to 2, of 1 up to 4, of 2 up to 6: half a step's tie goes to the even code
        code = torch.where(a < 2, (a * 2).round(), torch.where(a < 4, a.round() + 2, (a / 2).round() + 4)).clamp_max(7.0)
        code = (code.to(torch.uint8) | (torch.signbit(xf).to(torch.uint8) << 3)).flatten(-2)
        code = torch.where(s.repeat_interleave(16, -1) > 0, code, 0).unflatten(-1, (-1, 2))
        return code[..., 0] | (code[..., 1] << 4), (s.half().view(torch.int16) >> 7).to(torch.uint8)
    amax = xf.abs().amax(-1)
    top = torch.full_like(amax, MAXIMA[kind])
    inv = torch.where(amax > 0, top / amax, 0.0)
    y = xf * inv[..., None]
    codes = y.round().to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)
    return codes, amax / top


def _inv_freq(case):
    """Inverse frequencies [R / 2] in 64 bits, positions stretched evenly."""
    r = case["rotary_dim"]
    return 500000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r) / case["stretch"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = random.Random(seed)
    batch, heads, dim = case["batch"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rotary":
        # rows of each sequence follow what it holds; q and k are parts of one projection's output
        n = case["tokens"]
        cut = sorted(h.sample(range(1, n), batch - 1)) if batch > 1 else []
        at = []
        for a, e in zip([0] + cut, cut + [n]):
            start = h.randint(case["context"] // 2, case["context"])
            at += range(start, start + e - a)
        qkv = torch.randn((n, case["q_heads"] + 2 * heads, dim), generator=g, device="cuda", dtype=torch.float32)
        qkv = qkv.to(TYPES[case["type"]])
        return {"op": "rotary", "q": qkv[:, :case["q_heads"]], "k": qkv[:, case["q_heads"]:case["q_heads"] + heads],
                "positions": torch.tensor(at, dtype=torch.int32).cuda(), "inv_freq": _inv_freq(case).cuda(),
                "layout": case["layout"], "factor": case["factor"]}
    size = case["page"]
    counts, starts = _counts(case), _starts(case)
    need = [-(-(a + n) // size) for a, n in zip(starts, counts)]
    total = sum(need) + 3
    order = list(range(total))
    h.shuffle(order)
    table = torch.full((batch, max(need) + 2), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    shape = (total, heads, size, dim)
    k, v = _rows(case, shape, g), _rows(case, shape, g)
    s = {"op": case["op"], "type": case["type"], "page": size, "heads": heads, "dim": dim, "table": table.cuda(),
         "scale": dim ** -0.5, "k_scale": None, "v_scale": None, "rows": sum(counts), "longest": max(counts)}
    if case["type"] != "fp16":
        k, s["k_scale"] = _quantise(k, case["type"])
        v, s["v_scale"] = _quantise(v, case["type"])
    s["k"], s["v"] = k, v
    s["lens"] = torch.tensor(starts if case["op"] == "append" else counts, dtype=torch.int32).cuda()
    if case["op"] == "append":
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, dtype=torch.int32).cuda()
        s["one"] = case["tokens"] == 1 and not case["pad"]
        new = (s["rows"] + case["pad"], heads, dim)
        s["k_new"], s["v_new"] = _rows(case, new, g), _rows(case, new, g)
        return s
    if case["op"] in ("weigh", "evict"):
        # few positions carry most of the weight, some have had none
        w = torch.exp(2.0 * torch.randn(shape[:3], generator=g, device="cuda"))
        s["weight"] = torch.where(torch.rand(shape[:3], generator=g, device="cuda") < 0.03, 0.0, w)
    if case["op"] == "evict":
        s["keep"], s["first"], s["last"] = case["keep"], case["first"], case["last"]
    else:
        s["q"] = torch.randn((batch, case["q_heads"], dim), generator=g, device="cuda", dtype=torch.float16)
    return s


def run(s):
    return _own(s) if own else PLAIN[s["op"]](s)


def _own(s):
    from apple_amd import kernels as K

    if s["op"] == "rotary":
        q, k = K.rotary(s["q"], s["k"], s["positions"], s["inv_freq"], layout=s["layout"], factor=s["factor"])
        return {"q": q, "k": k}
    pages = K.KVPages(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["op"] == "append":
        K.paged_append(pages, s["table"], s["lens"], s["k_new"], s["v_new"], None if s["one"] else s["cu"])
        k, v = K.paged_read(pages, s["table"], s["lens"], s["cu"], s["rows"])
        return {"k": k, "v": v}
    if s["op"] == "attend":
        return {"out": K.paged_attention(s["q"], pages, s["table"], s["lens"], s["scale"])}
    if s["op"] == "weigh":
        out = K.paged_attention(s["q"], pages, s["table"], s["lens"], s["scale"], weight=s["weight"])
        return {"out": out, "weight": s["weight"]}
    # a copy of the weights, so that every pass on the same rows gives up the same positions
    weight = s["weight"].clone()
    lens = K.paged_evict(pages, s["table"], s["lens"], weight, s["keep"], first=s["first"], last=s["last"])
    return _pool(s) | {"weight": weight, "lens": lens}


def _pool(s):
    """The whole pool, codes as the bytes they are."""
    names = [n for n in ("k", "v", "k_scale", "v_scale") if s[n] is not None]
    return {n: s[n].view(torch.uint8) if s[n].dtype == torch.float8_e4m3fn else s[n] for n in names}


# ------------------------------------------------------------------ plain form

def _plain_rotary(s):
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = (torch.cos(angle) * s["factor"]).float()[:, None], (torch.sin(angle) * s["factor"]).float()[:, None]
    r = 2 * s["inv_freq"].shape[0]

    def turn(x):
        y = x.float()
        if s["layout"] == "half":
            a, b = y[..., :r // 2], y[..., r // 2:r]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([turned, y[..., r:]], -1).to(x.dtype)

    return {"q": turn(s["q"]), "k": turn(s["k"])}


def _places(s):
    """Page and row in the page of each of the call's rows."""
    n = torch.arange(s["rows"], device="cuda")
    cu = s["cu"].long()
    b = torch.searchsorted(cu[1:], n, right=True)
    pos = s["lens"].long()[b] + n - cu[b]
    return s["table"].long()[b, pos // s["page"]], pos % s["page"]


def _values(s, name, index):
    """Rows [..., D] in 32 bits at an index of page, head and row."""
    t, scale = s[name], s[name + "_scale"]
    if s["type"] == "fp16":
        return t[index].float()
    if s["type"] == "e2m1":
        code, step = t[index], (scale[index].short() << 7).view(torch.float16).float()
        code = torch.stack([code & 15, code >> 4], -1).flatten(-2).long()
        value = torch.tensor(E2M1 + [-x for x in E2M1], device="cuda")[code]
        return (value.unflatten(-1, (-1, 16)) * step[..., None]).flatten(-2)
    code = t[index] if s["type"] == "int8" else t.view(torch.uint8)[index].view(t.dtype)
    return code.float() * scale[index][..., None]


def _plain_append(s):
    page, row = _places(s)
    for name in ("k", "v"):
        s[name][page, :, row], s[name + "_scale"][page, :, row] = _quantise(s[name + "_new"][:s["rows"]], "e2m1")
    return {n: _values(s, n, (page, slice(None), row)).half() for n in ("k", "v")}


def _index(s):
    """Pages and rows of all positions, [B, longest], and whether they are the sequence's."""
    pos = torch.arange(s["longest"], device="cuda")
    page = s["table"].long()[:, pos // s["page"]]
    return page.clamp_min(0), (pos % s["page"]).expand(page.shape), pos < s["lens"][:, None]


def _plain_attend(s):
    page, row, there = _index(s)
    batch, q_heads, dim = s["q"].shape
    q = s["q"].float().view(batch, s["heads"], q_heads // s["heads"], dim)
    k, v = (_values(s, n, (page, slice(None), row)).transpose(1, 2) for n in ("k", "v"))  # [B, H, T, D]
    score = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    score = torch.where(there[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, torch.where(there[:, None, :, None], v, 0.0)) / total
    out = torch.where(total == 0, 0.0, out).reshape(s["q"].shape).half()
    if s["op"] == "attend":
        return {"out": out}
    p = torch.where(total == 0, 0.0, p / total).sum(2)                                    # [B, H, T]
    b, t = torch.nonzero(there, as_tuple=True)
    s["weight"][page[b, t], :, row[b, t]] += p[b, :, t]
    return {"out": out, "weight": s["weight"]}


def _plain_evict(s):
    weight = s["weight"].clone()
    page, row, there = _index(s)
    pos = torch.arange(s["longest"], device="cuda")
    lens = s["lens"].long()
    w = weight[page, :, row].transpose(1, 2)                                              # [B, H, T]
    always = (pos < s["first"]) | (pos >= lens[:, None] - s["last"])
    w = torch.where(always[:, None], math.inf, w.nan_to_num(math.inf, math.inf, -math.inf))
    w = torch.where(there[:, None], w, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :s["keep"]].sort(-1).values
    b = torch.nonzero(lens > s["keep"]).flatten()                                         # sequences that shrink
    if len(b):
        head = torch.arange(s["heads"], device="cuda")[None, :, None]
        old = (page[b][:, None].expand(-1, s["heads"], -1).gather(2, order[b]), head, order[b] % s["page"])
        new = torch.arange(s["keep"], device="cuda").expand(order[b].shape)
        to = (page[b][:, None, :s["keep"]].expand(new.shape), head, new % s["page"])
        for t in list(_pool(s).values()) + [weight]:
            t[to] = t[old]
    return _pool(s) | {"weight": weight, "lens": s["lens"].clamp_max(s["keep"])}


PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "weigh": _plain_attend,
         "evict": _plain_evict}


# ------------------------------------------------------------------ work and exact results

def work(case):
    heads, dim = case["kv_heads"], case["head_dim"]
    if case["op"] == "rotary":
        values = case["tokens"] * (case["q_heads"] + heads)
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": 2 * values * dim * size + 4 * case["tokens"] + 4 * case["rotary_dim"],
                "flops": 3 * values * case["rotary_dim"]}
    counts = _counts(case)
    row = {"fp16": 2 * dim, "int8": dim + 4, "e4m3": dim + 4, "e2m1": dim // 2 + dim // 16}[case["type"]]
    stored, plain = 2 * heads * row, 2 * heads * 2 * dim                                 # K and V of one token
    n = sum(counts)
    if case["op"] == "append":  # and read back
        return {"bytes": 2 * n * (plain + stored), "flops": 6 * n * heads * dim}
    if case["op"] == "evict":
        long = [m for m in counts if m > case["keep"]]
        moved = len(long) * (case["keep"] - case["first"])
        return {"bytes": sum(long) * heads * 4 + moved * (2 * stored + heads * 4), "flops": sum(long) * heads}
    moved = n * stored + case["batch"] * case["q_heads"] * dim * 2 * 2
    if case["op"] == "weigh":
        moved += 2 * n * heads * 4
    return {"bytes": moved, "flops": 4 * n * case["q_heads"] * dim}


def exact(case, seed):
    """Results in 64 bits, a sequence or a head at a time."""
    s = prepare(case, seed)
    if case["op"] == "rotary":
        r = case["rotary_dim"]
        turn = torch.polar(torch.full((1, 1), case["factor"], dtype=torch.float64, device="cuda"),
                           torch.outer(s["positions"].double(), s["inv_freq"]))[:, None]
        out = {}
        for name in ("q", "k"):
            x = s[name].double()
            first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            out[name] = x
        return out
    counts, starts = _counts(case), _starts(case)
    size, heads, dim = case["page"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        out = {}
        for name in ("k", "v"):
            x = s[name + "_new"][:s["rows"]].double().unflatten(-1, (-1, 16))
            scale = x.abs().amax(-1, keepdim=True) / 6
            unit = torch.exp2(torch.floor(torch.log2(scale.clamp_min(2.0 ** -14))) - 3)
            scale = torch.minimum((scale / unit).round() * unit, torch.tensor(10240.0, device="cuda"))
            y = torch.where(scale > 0, x / scale, 0.0).clamp(-6, 6)
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1.0))) - 1)  # one bit behind the leading one, from 1 up
            out[name] = ((y / step).round() * step * scale).flatten(-2)
        return out

    def rows(name, b, n):
        """[H, n, D] of sequence b."""
        ids = s["table"][b, :-(-n // size)].long()
        x = s[name]
        if case["type"] == "e2m1":
            raw = x[ids].long()
            parts = []
            for c in (raw % 16, raw // 16):
                e, m = (c % 8) // 2, c % 2
                parts.append(torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1))
                             * torch.where(c > 7, -1.0, 1.0).double())
            byte = s[name + "_scale"][ids].long()
            e, m = byte // 8, byte % 8
            unit = torch.where(e == 0, m / 8.0 * 2.0 ** -14, (1 + m / 8.0) * torch.exp2(e.double() - 15))
            x = torch.stack(parts, -1).flatten(-2) * unit.double().repeat_interleave(16, -1)
        elif case["type"] == "fp16":
            x = x[ids].double()
        else:
            x = (x.view(torch.uint8)[ids].view(x.dtype).float().double() if case["type"] == "e4m3" else x[ids].double())
            x = x * s[name + "_scale"][ids].double()[..., None]
        return x.transpose(0, 1).reshape(heads, -1, dim)[:, :n]

    if case["op"] in ("attend", "weigh"):
        outs, weight = [], s["weight"].double() if case["op"] == "weigh" else None
        for b, n in enumerate(counts):
            q = s["q"][b].double().view(heads, -1, dim)
            p = torch.softmax(torch.bmm(q, rows("k", b, n).transpose(1, 2).contiguous()) * s["scale"], -1)
            outs.append(torch.bmm(p, rows("v", b, n)).reshape(-1, dim))
            if weight is not None:
                held = -(-n // size)
                add = torch.nn.functional.pad(p.sum(1), (0, held * size - n)).view(heads, held, size)
                weight[s["table"][b, :held].long()] += add.transpose(0, 1)
        return {"out": torch.stack(outs)} | ({} if weight is None else {"weight": weight})
    pool = dict(_pool(s), weight=s["weight"])
    result = {name: t.clone() for name, t in pool.items()}
    for b, n in enumerate(counts):
        if n <= case["keep"]:
            continue
        ids = s["table"][b, :-(-n // size)].long()
        for h in range(heads):
            w = s["weight"][ids, h].flatten()[:n].double()
            w[:case["first"]] = w[n - case["last"]:] = math.inf
            kept = torch.sort(torch.argsort(-w, stable=True)[:case["keep"]]).values
            to = torch.arange(case["keep"], device="cuda")
            for name, t in pool.items():
                result[name][ids[to // size], h, to % size] = t[ids[kept // size], h, kept % size]
    return result | {"lens": torch.tensor([min(n, case["keep"]) for n in counts], dtype=torch.int32, device="cuda")}
