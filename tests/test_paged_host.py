"""The paged KV cache without a GPU: what its entry points refuse before a
launch, its workspace sizes, the parameter block's layout, and the cache's own
bookkeeping."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def lib():
    from apple_amd import _lib

    return _lib.load()


def block(**kw):
    """A parameter block whose addresses are never followed on the host."""
    from apple_amd import _lib

    p = _lib.Paged(k=4096, v=8192, table=16384, lens=20480, page_stride=8 * 16 * 64, head_stride=16 * 64,
                   table_stride=10, pages=5, page_size=16, kv_heads=8, head_dim=64, type=0, batch=2, table_width=10)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def test_parameter_block_layout(tmp_path):
    from apple_amd import _lib

    fields = [f for f, _ in _lib.Paged._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "rfsn_abi.h"\nint main(void) {\n'
                   'printf("size %zu\\n", sizeof(rfsn_paged));\n'
                   + "".join(f'printf("{f} %zu\\n", offsetof(rfsn_paged, {f}));\n' for f in fields) + "return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True,
                                                  check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(_lib.Paged)
    for f in fields:
        assert int(got[f]) == getattr(_lib.Paged, f).offset, f


def test_packed_block_is_the_parameter_block():
    """What the wrappers pack is the ctypes mirror's bytes."""
    from apple_amd import _lib
    from apple_amd.kernels import _PAGED_BLOCK

    values = [(i + 1) << 33 if ctypes.sizeof(t) == 8 else i + 1 for i, (_, t) in enumerate(_lib.Paged._fields_)]
    assert _PAGED_BLOCK.pack(*values) == bytes(_lib.Paged(*values))


@pytest.mark.parametrize("bad, says", [
    (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
    (dict(type=3), "page type"), (dict(kv_heads=0), "kv_heads"), (dict(batch=-1), "batch"), (dict(batch=70000), "batch"),
    (dict(pages=0), "no pages"), (dict(table_width=-1), "table"), (dict(table_width=1 << 28), "2^31"),
    (dict(table=0), "null table"), (dict(lens=0), "null lens"), (dict(k=0), "aligned"), (dict(v=8200), "aligned"),
    (dict(page_stride=8), "strides"), (dict(head_stride=64), "strides"), (dict(type=1), "scales"),
    (dict(k_scale=4096), "scales"), (dict(bounds=4100), "bounds must be")])
def test_pools_are_refused_before_a_launch(lib, bad, says):
    p = ctypes.byref(block(**bad))
    for name, args in (("rfsn_paged_append", (4096, 8192, 512, 64, 2, None, None)),
                       ("rfsn_paged_read", (4096, 2, 4096, 8192, 1, None)),
                       ("rfsn_page_select", (4096, 8, 4, 1, 1, 4096, 4096, 1 << 30, None)),
                       ("rfsn_paged_attention", (4096, 8, 0.125, None, 0, 4096, 4096, 1 << 30, None))):
        assert getattr(lib, name)(p, *args) == -1, name
        assert says.encode() in lib.rfsn_last_error(), (name, lib.rfsn_last_error())
        assert getattr(lib, name)(None, *args) == -1


@pytest.mark.parametrize("name, args, says", [
    ("rfsn_paged_append", (4096, 8192, 512, 64, -1, 4096, None), "row count"),
    ("rfsn_paged_append", (4096, 8192, 512, 64, 3, None, None), "one row per sequence"),
    ("rfsn_paged_append", (4098, 8192, 512, 64, 2, None, None), "aligned"),
    ("rfsn_paged_append", (4096, 8192, 510, 64, 2, None, None), "aligned"),
    ("rfsn_paged_append", (4096, 8192, 512, 64, 1 << 40, 4096, None), "too many rows"),
    ("rfsn_paged_read", (None, 2, 4096, 8192, 1, None), "null cu"),
    ("rfsn_paged_read", (4096, 2, 4096, 8200, 1, None), "aligned"),
    ("rfsn_paged_read", (4096, -2, 4096, 8192, 1, None), "row count"),
    ("rfsn_page_select", (4096, 8, 4, 1, 1, 4096, 4096, 1 << 30, None), "no bounds"),
    ("rfsn_paged_attention", (4096, 12, 0.125, None, 0, 4096, 4096, 1 << 30, None), "multiple of kv_heads"),
    ("rfsn_paged_attention", (4096, 8, 0.125, 4096, 0, 4096, 4096, 1 << 30, None), "together"),
    ("rfsn_paged_attention", (4096, 8, 0.125, None, 4, 4096, 4096, 1 << 30, None), "together"),
    ("rfsn_paged_attention", (4096, 8, 0.125, 4096, 1 << 29, 4096, 4096, 1 << 30, None), "too many chosen"),
    ("rfsn_paged_attention", (4096, 8, float("nan"), None, 0, 4096, 4096, 1 << 30, None), "finite"),
    ("rfsn_paged_attention", (4100, 8, 0.125, None, 0, 4096, 4096, 1 << 30, None), "aligned")])
def test_calls_are_refused_before_a_launch(lib, name, args, says):
    assert getattr(lib, name)(ctypes.byref(block()), *args) == -1
    assert says.encode() in lib.rfsn_last_error(), lib.rfsn_last_error()


@pytest.mark.parametrize("args, says", [
    ((4096, 12, 4, 1, 1, 4096, 4096, 1 << 30, None), "multiple of kv_heads"),
    ((4096, 8, 0, 0, 0, 4096, 4096, 1 << 30, None), "count"), ((4096, 8, 2, 2, 1, 4096, 4096, 1 << 30, None), "count"),
    ((4096, 8, 2, -1, 1, 4096, 4096, 1 << 30, None), "count"), ((4096, 8, 2, 1, 1, None, 4096, 1 << 30, None), "null"),
    ((4096, 8, 2, 1, 1, 4096, 4096, 8, None), "workspace")])
def test_selection_is_refused_before_a_launch(lib, args, says):
    assert lib.rfsn_page_select(ctypes.byref(block(bounds=4096)), *args) == -1
    assert says.encode() in lib.rfsn_last_error(), lib.rfsn_last_error()


@pytest.mark.parametrize("size", [16, 64, 256])
def test_page_counts_past_the_kernels_range_are_refused(lib, size):
    """The kernels step through a row of the list in 32-bit numbers: as many pages as positions below 2^31 hold, no more."""
    p = ctypes.byref(block(bounds=4096, page_size=size, page_stride=8 * size * 64, head_stride=size * 64))
    for count in (2 ** 31 - 1, 2 ** 31 - 512, 2 ** 31 // size):
        assert lib.rfsn_page_select(p, 4096, 8, count, 1, 1, 4096, 4096, 1 << 30, None) == -1
        assert b"too many pages" in lib.rfsn_last_error(), lib.rfsn_last_error()
        assert lib.rfsn_paged_attention(p, 4096, 8, 0.125, 4096, count, 4096, 4096, 1 << 30, None) == -1


def test_wrappers_refuse_page_counts_past_32_bits(monkeypatch):
    """ctypes would pass 2^32 + 4 pages on as 4."""
    from apple_amd import kernels as K

    monkeypatch.setattr(K, "_paged", lambda *a: (b"", (2, 2, 64, 16, 4), -1))
    monkeypatch.setattr(K, "_paged_call", lambda *a: pytest.fail("the call was made"))
    pages, table, lens = tensors()
    q = torch.zeros((2, 4, 64), dtype=torch.float16)
    for count in ((1 << 32) + 4, 1 << 31, (1 << 31) // 16):
        with pytest.raises(ValueError, match="pages of 16"):
            K.page_select(q, pages, table, torch.zeros(2, dtype=torch.int32, device="meta"), count)
        with pytest.raises(ValueError, match="pages of 16"):
            K.paged_attention(q, pages, table, lens, 0.1, torch.zeros((1, 1, 1), dtype=torch.int32).expand(2, 2, count))


def test_workspace_sizes(lib):
    size = lib.rfsn_paged_attention_workspace_bytes
    assert size(None, 8, 0) == 0
    assert size(ctypes.byref(block()), 8, 0) == 0  # 160 positions: one chunk, no partials
    wide = block(table_width=4096)
    need = size(ctypes.byref(wide), 32, 0)
    assert need > 32 * 66 * 4  # partial results of several chunks
    assert lib.rfsn_paged_attention(ctypes.byref(wide), 4096, 32, 0.125, None, 0, 4096, 4096, need - 1, None) == -1
    assert b"workspace" in lib.rfsn_last_error()
    assert lib.rfsn_page_select_workspace_bytes(ctypes.byref(wide)) >= 2 * 8 * 4096 * 4
    # an empty batch is no error and launches nothing
    none = ctypes.byref(block(batch=0, table=0, lens=0))
    assert lib.rfsn_paged_attention(none, None, 8, 0.125, None, 0, None, None, 0, None) == 0
    assert lib.rfsn_paged_append(none, None, None, 0, 0, 0, None, None) == 0


def tensors(kind=torch.float16, batch=2):
    from apple_amd.kernels import KVPages

    k = torch.zeros((4, 2, 16, 64), dtype=kind)
    s = None if kind == torch.float16 else torch.zeros((4, 2, 16))
    return (KVPages(k, k.clone(), s, s, torch.zeros((4, 2, 2, 64), dtype=torch.float16)),
            torch.zeros((batch, 4), dtype=torch.int32), torch.zeros(batch, dtype=torch.int32))


def test_host_tensors_are_refused():
    from apple_amd import kernels as K

    pages, table, lens = tensors()
    q = torch.zeros((2, 4, 64), dtype=torch.float16)
    for call in (lambda: K.paged_attention(q, pages, table, lens, 0.125),
                 lambda: K.page_select(q, pages, table, lens, 2),
                 lambda: K.paged_append(pages, table, lens, q[:, :2], q[:, :2]),
                 lambda: K.paged_read(pages, table, lens, torch.zeros(3, dtype=torch.int32), 0)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def config(**kw):
    from apple_amd.storage import RFSNConfig

    return RFSNConfig(**{**dict(hidden_dim=512, num_heads=8, num_kv_heads=2, head_dim=64, num_subspaces=8,
                                subspace_dim=8), **kw})


def test_cache_arguments():
    from apple_amd.paged import RFSNPagedKVCache

    make = lambda **kw: RFSNPagedKVCache(config(), **{**dict(batch=2, pages=8, device="cpu"), **kw})
    for bad in (dict(batch=0), dict(pages=0), dict(page_size=24), dict(page_type="bf16"), dict(max_tokens=0)):
        with pytest.raises(ValueError):
            make(**bad)
    with pytest.raises(ValueError):
        RFSNPagedKVCache(config(head_dim=32, num_subspaces=8, subspace_dim=4), 2, 8, device="cpu")
    assert make().table.shape == (2, 8)
    assert make(max_tokens=100).table.shape == (2, 2) and make(max_tokens=100).max_tokens == 100
    assert make(bounds=False).pages.bounds is None


def test_cache_page_bookkeeping(monkeypatch):
    """Pages are taken when a sequence passes its last one's end and return on release; a refused call takes none."""
    from apple_amd import kernels as K
    from apple_amd.paged import RFSNPagedKVCache

    calls = []
    monkeypatch.setattr(K, "paged_append", lambda pages, table, lens, k, v, cu=None: calls.append(
        (lens.clone(), None if cu is None else cu.clone())))
    c = RFSNPagedKVCache(config(), batch=3, pages=5, page_size=16, max_tokens=64, device="cpu")
    rows = lambda n: torch.zeros((n, 2, 64), dtype=torch.float16)
    c.append(rows(20), rows(20), [16, 0, 4])
    assert c.free_pages == 3 and c.num_tokens == [16, 0, 4] and c.lens.tolist() == [16, 0, 4]
    assert calls[-1][0].tolist() == [0, 0, 0] and calls[-1][1].tolist() == [0, 16, 16, 20]
    c.append(rows(3), rows(3))
    assert calls[-1][1] is None and c.lens.tolist() == [17, 1, 5] and c.free_pages == 1
    held = c.table[c.table >= 0].tolist()
    assert len(set(held)) == len(held) == 4
    for bad, error in ((lambda: c.append(rows(2), rows(2)), ValueError), (lambda: c.prefill(3, rows(1), rows(1)), ValueError),
                       (lambda: c.append(rows(3), rows(2)), ValueError), (lambda: c.prefill(1, rows(64), rows(64)), ValueError),
                       (lambda: c.append(rows(3), rows(3), [4, -1, 0]), ValueError),
                       (lambda: c.append(rows(40), rows(40), [0, 20, 20]), RuntimeError),
                       (lambda: c.attention_forward(torch.zeros((2, 8, 64))), ValueError),
                       (lambda: c.attention_forward(torch.zeros((3, 8, 64)), sparse_pages=1), ValueError),
                       (lambda: c.prompt_attention(2, torch.zeros((6, 8, 64))), ValueError)):
        with pytest.raises(error):
            bad()
    assert c.free_pages == 1 and c.num_tokens == [17, 1, 5] and c.lens.tolist() == [17, 1, 5]
    c.release(0)
    assert c.free_pages == 3 and c.num_tokens == [0, 1, 5] and c.table[0].tolist() == [-1] * 4
    assert c.lens.tolist() == [0, 1, 5]
    use = c.memory_usage_bytes()
    assert use["in_use"] * 5 == use["pool"] * 2 > 0


def test_cache_steps_after_a_release(monkeypatch):
    """A step without counts gives a released sequence no token: it is refused until a successor holds some, and takes
    no page; a step of a batch that is released as a whole starts all of it again."""
    from apple_amd import kernels as K
    from apple_amd.paged import RFSNPagedKVCache

    monkeypatch.setattr(K, "paged_append", lambda pages, table, lens, k, v, cu=None: None)
    c = RFSNPagedKVCache(config(), batch=3, pages=6, page_size=16, device="cpu")
    rows = lambda n: torch.zeros((n, 2, 64), dtype=torch.float16)
    step = lambda *counts: c.append(rows(sum(counts) if counts else 3), rows(sum(counts) if counts else 3), counts or None)
    step(5, 0, 7)
    step()  # the second was never begun: it starts here
    assert c.num_tokens == [6, 1, 8]
    c.release(1)
    for held in ([6, 0, 8], [7, 0, 9]):
        with pytest.raises(ValueError, match=r"sequences \[1\] were released"):
            step()
        assert c.num_tokens == held == c.lens.tolist() and c.free_pages == 4 and c.table[1].tolist() == [-1] * 6
        step(1, 0, 1)
    c.prefill(1, rows(4), rows(4))
    step()
    assert c.num_tokens == [9, 5, 11]
    for b in range(3):
        c.release(b)
    step()  # all of them begin
    assert c.num_tokens == [1, 1, 1]
    c.release(2)
    c.release(0)
    with pytest.raises(ValueError, match=r"\[0, 2\]"):
        step()
    step(1, 1, 0)
    with pytest.raises(ValueError, match=r"\[2\]"):
        step()
    step(0, 0, 1)
    step()
    assert c.num_tokens == [2, 3, 2]


def test_reference_quantiser_round_trip():
    """The host restatement itself: a value comes back within half a code step."""
    from tests.paged_reference import quantise

    g = torch.Generator().manual_seed(3)
    x = (torch.randn((50, 64), generator=g) * torch.rand((50, 1), generator=g) * 30).half()
    x[7] = 0
    for dtype, step in ((torch.int8, None), (torch.float8_e4m3fn, 2.0 ** -4)):
        codes, scale = quantise(x, dtype)
        back = codes.float() * scale[:, None]
        half = scale[:, None] * 0.5 if step is None else torch.maximum(x.float().abs() * step, scale[:, None] * 2.0 ** -10)
        assert ((back - x.float()).abs() <= half * (1 + 1e-5)).all()
        assert (codes[7].float() == 0).all() and scale[7] == 0


@pytest.mark.parametrize("kind", ["fp16", "int8", "e4m3"])
def test_what_a_page_s_score_says_of_its_keys(kind):
    """No q . k of the keys as they were appended exceeds the page's score; what is attended of an 8-bit page may, by half a
    code step per coordinate: int8 stores 0.6 beside 127 as 1."""
    from tests import paged_reference as R

    g = torch.Generator().manual_seed(5)
    over = 0
    for trial in range(60):
        rows = 1 if trial % 2 else 16
        k = torch.randn((rows, 64), generator=g).half()
        q = torch.randn(64, generator=g).half()
        if trial == 1:  # values that round up: 0.6 to 1, and 1.07 to 1.125 (e4m3 turns at 1.0625)
            k[0], q[:] = 0, 0
            k[0, 0], k[0, 1], q[1] = (127.0, 0.6, 8.0) if kind == "int8" else (448.0, 1.07, 8.0)
        pool = R.Pool(kind, 1, 1, 16, 64, seed=1)
        pool.append(torch.zeros((1, 1), dtype=torch.int32), [0], k[:, None], k[:, None], [0, rows])
        lo, hi = pool.bounds[0, 0].double()
        x = q.double()
        score = float((x.clamp(min=0) * hi + x.clamp(max=0) * lo).sum().float())
        slack = 2.0 ** -24 * abs(score)  # the score's rounding to fp32
        assert float((k.double() @ x).max()) <= score + slack
        held = pool.values("k")[0, 0, :rows]
        if kind == "fp16":
            assert torch.equal(held, k.double())
            continue
        scale = pool.k_scale[0, 0, :rows].double()[:, None]
        half = scale / 2 if kind == "int8" else torch.maximum(k.double().abs() * 2.0 ** -4, scale * 2.0 ** -10)
        # the quantiser's own product and reciprocal are off by 2^-22 of the value
        more = ((half + k.double().abs() * 2.0 ** -22) * x.abs()).sum(-1)
        assert (held @ x <= score + slack + more).all()
        over += bool((held @ x > score + slack).any())
        if trial == 1:
            assert float((held @ x)[0]) > score + 0.1
    assert over > 0 or kind == "fp16"


# ------------------------------------------------------------------ the plan of an attention call

@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """(slots, wide, once, chunks per sequence, chunk) of a call, from the host's own source."""
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cc").write_text('''#include "paged_plan.h"
extern "C" void plan_of(const rfsn_paged* p, int q_heads, int count, int64_t* out, float* one_over) {
  const rfsn::Plan r = rfsn::plan(*p, q_heads, count);
  out[0] = r.slots, out[1] = r.wide, out[2] = r.once, out[3] = r.cut.per_seq, out[4] = r.cut.chunk, out[5] = r.cut.longest;
  for (int x = 0; x < rfsn::kTries; ++x) one_over[x] = r.cut.one_over[x];
}
''')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{ROOT / 'include'}",
                    f"-I{ROOT / 'apple_amd' / 'csrc'}", str(at / "plan.cc"), "-o", str(at / "plan.so")], check=True)
    fn = ctypes.CDLL(str(at / "plan.so")).plan_of

    def call(q_heads, count=0, **kw):
        out, one_over = (ctypes.c_int64 * 6)(), (ctypes.c_float * 3)()
        fn(ctypes.byref(block(**kw)), q_heads, count, out, one_over)
        return dict(zip(("slots", "wide", "once", "per_seq", "chunk", "longest"), out), one_over=list(one_over))

    return call


def test_rows_count_as_used_once_by_what_is_read(plan):
    """256 MB of pages that a call reads, not of pages that there are or that wide tables could name."""
    # a pool of 4 GB: 2 MB of K and V a page with 8 heads of 256
    pool = dict(pages=2048, page_size=256, kv_heads=8, head_dim=256)
    for batch, width, held, once in ((64, 5, 0, True), (65, 2, 0, True), (64, 8, 127, False), (64, 8, 128, True),
                                     (64, 8, 1 << 30, True), (64, 2048, 100, False), (64, 2048, 0, True)):
        assert plan(32, batch=batch, table_width=width, table_stride=width, held_pages=held, **pool)["once"] == once
    # many queries over one sequence's pages: one row of the table for all of them
    for width, once in ((32, False), (127, False), (128, True)):
        assert plan(32, batch=512, table_width=width, table_stride=0, **pool)["once"] == once
        assert plan(32, batch=512, table_width=width, table_stride=width, **pool)["once"]
    # a list of pages, and blocks of many waves, are never loaded so
    assert not plan(32, count=16, batch=64, table_width=64, table_stride=64, **pool)["once"]


def test_a_hint_changes_nothing_but_how_rows_are_loaded(plan, lib):
    for kw in (dict(batch=48, table_width=250, page_size=64, kv_heads=4), dict(batch=1, table_width=4096, kv_heads=8),
               dict(batch=600, table_width=600, kv_heads=2)):
        a, b = (plan(32, pages=1 << 20, held_pages=n, **kw) for n in (0, 3))
        a.pop("once"), b.pop("once")
        assert a == b
        sizes = [lib.rfsn_paged_attention_workspace_bytes(ctypes.byref(block(pages=1 << 20, held_pages=n, **kw)), 32, 0)
                 for n in (0, 3)]
        assert sizes[0] == sizes[1] > 0


def chunks_by_lengths(cut, lens):
    """Chunks of each sequence for each size that the device may choose, and the longest of them: find_chunk's arithmetic
    in fp32."""
    f = torch.float32
    for one_over in cut["one_over"]:
        each = torch.tensor(sum(lens), dtype=f) * torch.tensor(one_over, dtype=f) + torch.tensor(0.98, dtype=f)
        size = min(int(each), 2147483520)
        size = cut["chunk"] if size <= cut["chunk"] else (size + 127) // 128 * 128
        size = min(size, cut["longest"])
        n = [-(-t // size) for t in lens]
        yield sum(n), max((-(-(-(-t // m)) // 128) * 128 for t, m in zip(lens, n) if m), default=0)


def test_every_chunk_has_a_slot_and_none_is_too_long(plan):
    """Batches of one to many sequences, alike and ragged, up to the capacity's limit."""
    import random

    rng = random.Random(7)
    seen = 0
    for i in range(600):
        batch = rng.choice([1, 1, 2, 3, 31, 64, 65, 500, 4000, 32000])
        size = rng.choice([16, 64, 256])
        most = 2 ** 31 - 1024 if i % 4 == 0 else int(2 ** rng.uniform(7, 30.9))
        heads, group, dim = rng.choice([1, 2, 8, 32, 512, 3000]), rng.choice([1, 4, 20]), rng.choice([64, 128, 256])
        width = max(1, most // size)
        cut = plan(heads * group, batch=batch, table_width=width, table_stride=width, page_size=size, kv_heads=heads, head_dim=dim)
        assert cut["longest"] >= 1 << 22
        assert cut["longest"] == 1 << 22 or (cut["longest"] // 2 < width * size and
                                             -(-width * size // (cut["longest"] // 2)) * batch > 32768)
        if cut["per_seq"]:
            assert cut["per_seq"] == 1 and cut["slots"] == batch and cut["chunk"] == width * size <= 4096
            continue
        seen += 1
        lens = [width * size if rng.random() < 0.5 else int((width * size) ** rng.random()) for _ in range(min(batch, 500))]
        lens = (lens * -(-batch // len(lens)))[:batch]
        for all_of in (lens, [width * size] * batch, [0] * (batch - 1) + [width * size]):
            for chunks, longest in chunks_by_lengths(cut, all_of):
                assert chunks <= cut["slots"] and longest <= max(cut["longest"], cut["chunk"]), (cut, chunks, longest)
        if batch <= 4000:
            assert cut["slots"] <= 65535
    assert seen > 200


def test_lists_of_pages_are_cut_below_the_longest_chunk(plan):
    for batch, heads, count, size in ((1, 512, 1 << 19, 64), (3, 700, (1 << 31) // 16 - 64, 16), (1, 1, 1 << 22, 256), (64, 8, 128, 16),
                                      (2000, 4, 1 << 18, 256), (40000, 1, 1 << 20, 64), (512, 8, 1 << 16, 256)):
        cut = plan(heads, count, batch=batch, table_width=1 << 20, page_size=size, kv_heads=heads)
        assert cut["per_seq"] * cut["chunk"] >= count * size and cut["slots"] == cut["per_seq"] * batch <= 65535
        assert (cut["per_seq"] - 1) * cut["chunk"] < count * size
        assert cut["chunk"] <= cut["longest"] and (cut["longest"] == 1 << 22 or batch > 64)


def test_cache_says_what_it_holds(monkeypatch):
    from apple_amd import kernels as K
    from apple_amd.paged import RFSNPagedKVCache

    said = []
    monkeypatch.setattr(K, "paged_append", lambda *a: None)
    monkeypatch.setattr(K, "paged_attention", lambda q, pages, table, lens, scale, chosen=None, held_pages=0:
                        said.append((held_pages, table.stride(0))) or q)
    c = RFSNPagedKVCache(config(), batch=2, pages=20, page_size=16, device="cpu")
    rows = torch.zeros((60, 2, 64), dtype=torch.float16)
    c.append(rows, rows, [35, 25])
    c.attention_forward(torch.zeros((2, 8, 64)))
    wide = RFSNPagedKVCache(config(head_dim=256, subspace_dim=32), batch=2, pages=20, page_size=16, device="cpu")
    rows = torch.zeros((60, 2, 256), dtype=torch.float16)
    wide.append(rows, rows, [35, 25])
    wide.prompt_attention(0, torch.zeros((7, 8, 256)))
    assert said == [(5, 20), (0, 0)]  # two tables of 3 and 2 pages; one row for all queries of a chunk
