"""What bounds a paged cache's memory, without a GPU: what the entry points
refuse before a launch, the parameter blocks' layout, the restatement's own
properties, and the cache's bookkeeping."""

import ctypes
import math
import subprocess

import pytest
import torch

from tests import bounded_reference as B
from tests.test_paged_host import ROOT, block, chunks_by_lengths, config, lib, plan  # noqa: F401


def four(**kw):
    return block(**{**dict(type=4, k_scale=4096, v_scale=4096, page_stride=8 * 16 * 64, head_stride=16 * 64), **kw})


def test_rotary_block_layout(tmp_path):
    from apple_amd import _lib

    fields = [f for f, _ in _lib.RotaryParams._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "rfsn_abi.h"\nint main(void) {\n'
                   'printf("size %zu\\n", sizeof(rfsn_rotary_params));\n'
                   + "".join(f'printf("{f} %zu\\n", offsetof(rfsn_rotary_params, {f}));\n' for f in fields) + "return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(_lib.RotaryParams)
    for f in fields:
        assert int(got[f]) == getattr(_lib.RotaryParams, f).offset, f


def test_packed_rotary_block_is_the_parameter_block():
    from apple_amd import _lib
    from apple_amd.kernels import _ROTARY_BLOCK

    p, flat = _lib.RotaryParams(), []
    for n, (name, t) in enumerate(_lib.RotaryParams._fields_):
        if hasattr(t, "_length_"):
            values = [(100 * n + i) for i in range(2)]
            setattr(p, name, t(*values))
            flat += values
        else:
            setattr(p, name, n + 1)
            flat.append(n + 1)
    assert _ROTARY_BLOCK.pack(*flat) == bytes(p)


def test_four_bit_pools_are_refused_before_a_launch(lib):
    for bad, says in ((dict(k_scale=0), "scales"), (dict(v_scale=0), "scales"), (dict(head_stride=16 * 64 + 16), "strides"),
                      (dict(page_stride=8 * 16 * 64 + 16), "strides"), (dict(weight=4100), "weights must be")):
        p = ctypes.byref(four(**bad))
        for name, args in (("rfsn_paged_append", (4096, 8192, 512, 64, 2, None, None)),
                           ("rfsn_paged_read", (4096, 2, 4096, 8192, 1, None)),
                           ("rfsn_paged_evict", (16, 4, 4, 4096, 4096, 1 << 30, None)),
                           ("rfsn_paged_attention", (4096, 8, 0.125, None, 0, 4096, 4096, 1 << 30, None))):
            assert getattr(lib, name)(p, *args) == -1, name
            assert says.encode() in lib.rfsn_last_error(), (name, lib.rfsn_last_error())


@pytest.mark.parametrize("args, says", [
    ((0, 0, 0, 4096, 4096, 1 << 30, None), "keep"), ((-5, 0, 0, 4096, 4096, 1 << 30, None), "keep"),
    ((16, 9, 8, 4096, 4096, 1 << 30, None), "keep"), ((16, -1, 8, 4096, 4096, 1 << 30, None), "keep"),
    ((16, 0, -8, 4096, 4096, 1 << 30, None), "keep"), ((16, 4, 4, None, 4096, 1 << 30, None), "null output"),
    ((16, 2 ** 31 - 1, 2 ** 31 - 1, 4096, 4096, 1 << 30, None), "keep"),
    ((16, 4, 4, 4096, None, 1 << 30, None), "workspace"), ((16, 4, 4, 4096, 4096, 2 * 8 * 16 * 4 - 1, None), "workspace")])
def test_evictions_are_refused_before_a_launch(lib, args, says):
    assert lib.rfsn_paged_evict(ctypes.byref(block(weight=4096)), *args) == -1
    assert says.encode() in lib.rfsn_last_error(), lib.rfsn_last_error()
    assert lib.rfsn_paged_evict(None, *args) == -1


def test_weights_go_with_whole_sequences(lib):
    assert lib.rfsn_paged_evict(ctypes.byref(block()), 16, 4, 4, 4096, 4096, 1 << 30, None) == -1
    assert b"no weights" in lib.rfsn_last_error()
    assert lib.rfsn_paged_attention(ctypes.byref(block(weight=4096)), 4096, 8, 0.125, 4096, 4, 4096, 4096, 1 << 30, None) == -1
    assert b"chosen pages" in lib.rfsn_last_error()
    size = lib.rfsn_paged_attention_workspace_bytes
    # scores of 160 positions and (m, l) of 8 query heads, two sequences
    assert size(ctypes.byref(block(weight=4096)), 8, 0) == 2 * 8 * (160 + 2) * 4 + size(ctypes.byref(block()), 8, 0)
    wide = block(table_width=4096, weight=4096)
    need = size(ctypes.byref(wide), 32, 0)
    assert need >= 2 * 32 * 4096 * 16 * 4 + size(ctypes.byref(block(table_width=4096)), 32, 0)
    assert lib.rfsn_paged_attention(ctypes.byref(wide), 4096, 32, 0.125, None, 0, 4096, 4096, need - 1, None) == -1
    assert b"workspace" in lib.rfsn_last_error()
    # an empty batch is no error and launches nothing
    none = ctypes.byref(block(batch=0, table=0, lens=0, weight=4096))
    assert lib.rfsn_paged_evict(none, 16, 4, 4, None, None, 0, None) == 0
    assert lib.rfsn_paged_attention(none, None, 8, 0.125, None, 0, None, None, 0, None) == 0


def test_four_bit_chunks_have_slots_in_a_workspace_that_knows_no_type(plan, lib):
    import random

    rng = random.Random(9)
    codes = dict(type=4, k_scale=4096, v_scale=4096)
    seen = 0
    for i in range(500):
        batch, size = rng.choice([1, 2, 17, 24, 64, 65, 500, 4000, 4097, 20000, 32000]), rng.choice([16, 64, 256])
        heads, group, dim = rng.choice([1, 2, 8, 32, 512]), rng.choice([1, 4, 20]), rng.choice([64, 128, 256])
        width = max(1, int(2 ** rng.uniform(7, 24)) // size)
        kw = dict(batch=batch, table_width=width, table_stride=width, page_size=size, kv_heads=heads, head_dim=dim,
                  head_stride=size * dim, page_stride=heads * size * dim)
        cut = plan(heads * group, **codes, **kw)
        assert cut["slots"] == plan(heads * group, **kw)["slots"] <= 65535
        sizes = [lib.rfsn_paged_attention_workspace_bytes(ctypes.byref(block(**of, **kw)), heads * group, 0) for of in (codes, {})]
        assert sizes[0] == sizes[1]
        if cut["per_seq"]:
            continue
        seen += 1
        lens = [width * size if rng.random() < 0.5 else int((width * size) ** rng.random()) for _ in range(min(batch, 300))]
        lens = (lens * -(-batch // len(lens)))[:batch]
        for all_of in (lens, [width * size] * batch, [0] * (batch - 1) + [width * size]):
            for chunks, longest in chunks_by_lengths(cut, all_of):
                assert chunks <= cut["slots"] and longest <= max(cut["longest"], cut["chunk"]), (cut, chunks, longest)
    assert seen > 150


def test_weights_of_sequences_that_share_a_table_are_refused(lib):
    shared = block(weight=4096, table_stride=0)
    assert lib.rfsn_paged_attention(ctypes.byref(shared), 4096, 8, 0.125, None, 0, 4096, 4096, 1 << 30, None) == -1
    assert b"share a table" in lib.rfsn_last_error()
    assert lib.rfsn_paged_evict(ctypes.byref(shared), 16, 4, 4, 4096, 4096, 1 << 30, None) == -1
    assert b"share a table" in lib.rfsn_last_error()


def test_rotary_calls_are_refused_before_a_launch(lib):
    from apple_amd import _lib

    def call(**kw):
        p = _lib.RotaryParams(rows=3, head_dim=64, rotary_dim=64, layout=0, type=0, positions=4096, inv_freq=4096, factor=1.0)
        p.heads[0], p.heads[1] = 8, 2
        for i in range(2):
            p.x[i], p.out[i] = 4096, 8192
        for name, value in kw.items():
            setattr(p, name, value)
        return lib.rfsn_rotary(ctypes.byref(p), None)

    for bad, says in ((dict(head_dim=1), "head_dim"), (dict(head_dim=2048), "head_dim"), (dict(rotary_dim=0), "rotary_dim"),
                      (dict(rotary_dim=66), "rotary_dim"), (dict(rotary_dim=7), "rotary_dim"), (dict(layout=2), "layout"),
                      (dict(type=3), "type"), (dict(rows=-1), "row count"), (dict(rows=1 << 31), "row count"),
                      (dict(positions=None), "positions"), (dict(positions=4098), "positions"),
                      (dict(positions=4100, wide_positions=1), "positions"), (dict(inv_freq=4100), "frequencies"),
                      (dict(heads=(ctypes.c_int32 * 2)(-1, 2)), "heads"), (dict(x=(ctypes.c_void_p * 2)(4097, 4096)), "rows"),
                      (dict(out=(ctypes.c_void_p * 2)(4096, None)), "rows"), (dict(x=(ctypes.c_void_p * 2)(4096, 4098), type=2), "rows")):
        assert call(**bad) == -1, bad
        assert says.encode() in lib.rfsn_last_error(), (bad, lib.rfsn_last_error())
    assert lib.rfsn_rotary(None, None) == -1
    assert call(rows=0) == 0 and call(heads=(ctypes.c_int32 * 2)(0, 0)) == 0


def test_wrappers_refuse_host_tensors():
    from apple_amd import kernels as K
    from tests.test_paged_host import tensors

    pages, table, lens = tensors()
    w = torch.zeros((4, 2, 16))
    q = torch.zeros((2, 4, 64), dtype=torch.float16)
    for call in (lambda: K.paged_evict(pages, table, lens, w, 8), lambda: K.paged_attention(q, pages, table, lens, 0.1, weight=w),
                 lambda: K.rotary(q, None, lens, torch.ones(32, dtype=torch.float64))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(ValueError, match="chosen pages"):
        K.paged_attention(q, pages, table, lens, 0.1, torch.zeros((2, 2, 1), dtype=torch.int32), weight=w)


def test_memory_that_rows_share():
    """Which tensors may be turned in place."""
    from apple_amd.kernels import _apart, _clear_of

    wide = torch.zeros((5, 12, 64))
    q, k = wide[:, :8], wide[:, 8:10]
    assert _apart(q) and _apart(k) and _clear_of(q, k) and _clear_of(k, q)
    assert not _clear_of(q, q) and not _clear_of(q, wide[:, 7:9]) and _clear_of(q, torch.zeros((5, 2, 64)))
    assert not _apart(torch.zeros((1, 8, 64)).expand(5, 8, 64)) and not _apart(torch.zeros((5, 1, 64)).expand(5, 8, 64))
    assert not _apart(wide.as_strided((5, 8, 64), (32, 256, 1))) and _apart(wide.as_strided((5, 8, 64), (64, 320, 1)))
    assert _apart(wide[:, :, :32]) and _apart(wide[:1].expand(1, 12, 64)) and not _clear_of(wide[:, :, :32], wide[:, :, 32:])
    assert _clear_of(wide[:2], wide[2:4]) and not _clear_of(wide[:3], wide[2:5])


def test_four_bit_quantiser_of_the_restatement():
    """Its values are the nearest that there are, its scales the numbers that the format names."""
    assert torch.isnan(B.SCALES[249:]).all() and B.SCALES[248] == math.inf and B.SCALES[B.TOP] == 10240
    assert B.SCALES[1] == 2.0 ** -17 and B.SCALES[8] == 2.0 ** -14 and B.SCALES[120] == 1.0 and B.SCALES[121] == 1.125
    g = torch.Generator().manual_seed(3)
    x = (torch.randn((200, 64), generator=g) * torch.exp2(torch.randint(-14, 12, (200, 1), generator=g).float())).half()
    codes, scales = B.quantise4(x)
    back = B.values4(codes, scales)
    assert torch.equal(back.half().double(), back)  # exact in fp16
    step = B.SCALES[scales.long()].repeat_interleave(16, -1)
    every = torch.cat([B.MAGNITUDES, -B.MAGNITUDES])
    best = (x.double()[..., None] - every * step[..., None]).abs().amin(-1)
    assert torch.equal((x.double() - back).abs(), best)
    # the largest of a group is off by at most a sixth of itself (the step between 4 and 6) and the scale's half step,
    # or half a step of the smallest scales
    top = x.abs().double().unflatten(-1, (-1, 16)).amax(-1)
    off = ((x.double() - back).abs().unflatten(-1, (-1, 16)).amax(-1) - top * (1 / 6 + 2.0 ** -4)).amax()
    assert float(off) <= 6 * 2.0 ** -18


def test_four_bit_quantiser_of_the_timed_cases():
    import importlib.util

    spec = importlib.util.spec_from_file_location("more_operators", ROOT / "perf" / "more_operators.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    g = torch.Generator().manual_seed(4)
    x = (torch.randn((300, 64), generator=g) * torch.exp2(torch.randint(-16, 12, (300, 1), generator=g).float())).half()
    x[0], x[1, :16] = 0, 1e-6
    codes, scales = m._quantise(x, "e2m1")
    want = B.quantise4(x)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])


def test_cache_keeps_account_of_what_is_given_up(monkeypatch):
    """Pages return, positions go on, and a prompt chunk may not pass a gap."""
    from apple_amd import kernels as K
    from apple_amd.paged import RFSNPagedKVCache

    calls = []
    monkeypatch.setattr(K, "paged_append", lambda pages, table, lens, k, v, cu=None, weight=None: calls.append(weight))
    monkeypatch.setattr(K, "paged_evict", lambda pages, table, lens, weight, keep, *, first, last: lens.clamp_max(keep))
    monkeypatch.setattr(K, "paged_attention", lambda q, *a, weight=None: calls.append(weight) or q)
    monkeypatch.setattr(K, "page_select", lambda *a: torch.zeros((3, 2, 2), dtype=torch.int32))
    c = RFSNPagedKVCache(config(), batch=3, pages=20, page_size=16, page_type="e2m1", device="cpu", weights=True)
    assert c.pages.k.shape == (20, 2, 16, 32) and c.pages.k_scale.shape == (20, 2, 16, 4) and c.weight.shape == (20, 2, 16)
    use = c.memory_usage_bytes()
    assert use["weights"] == 20 * 2 * 16 * 4 and use["pool"] == 20 * 2 * (16 * (64 + 8) + 2 * 64 * 2)
    rows = lambda n: torch.zeros((n, 2, 64), dtype=torch.float16)
    assert c.positions([2, 0, 1]).tolist() == [0, 1, 0]
    c.append(rows(150), rows(150), [100, 20, 30])
    assert calls[-1] is c.weight and c.free_pages == 20 - 7 - 2 - 2
    c.attention_forward(torch.zeros((3, 8, 64)))
    assert calls[-1] is c.weight
    c.attention_forward(torch.zeros((3, 8, 64)), sparse_pages=2)
    assert calls[-1] is None
    for bad in ((0, 0, 0), (10, 6, 5), (10, -1, 5), (10, 1, -5)):
        with pytest.raises(ValueError):
            c.evict(*bad)
    c.evict(100)
    assert c.num_tokens == [100, 20, 30] and c.free_pages == 9
    c.evict(25, 2, 10)
    assert c.num_tokens == [25, 20, 25] == c.lens.tolist() and c.free_pages == 9 + 5
    assert (c.table[0, 2:] == -1).all() and (c.table[:, :2] >= 0).all()
    held = c.table[c.table >= 0].tolist() + c._free
    assert len(set(held)) == len(held) == 20
    assert c.positions().tolist() == [100, 20, 30]
    c.append(rows(3), rows(3))
    assert c.positions().tolist() == [101, 21, 31] and c.positions([0, 2, 1]).tolist() == [21, 22, 31]
    for b, most in ((0, 11), (1, 21), (2, 11)):
        with pytest.raises(ValueError, match="gap" if b != 1 else "held"):
            c.prompt_attention(b, torch.zeros((most + 1, 8, 64)))
    c.evict(22, 0, 20)  # the 20 newest rows of the first are 11 newest tokens and some before a gap
    assert c._gaps == [11, 0, 11] and c.num_tokens == [22, 21, 22]
    c.release(0)
    assert c.positions().tolist() == [0, 21, 31] and c._gaps[0] == 0
    with pytest.raises(ValueError):
        c.positions([1, 2])
    plain = RFSNPagedKVCache(config(), batch=1, pages=4, page_size=16, device="cpu")
    with pytest.raises(ValueError, match="weights=True"):
        plain.evict(10)
    assert plain.weight is None and "weights" not in plain.memory_usage_bytes()
