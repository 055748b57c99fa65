"""A paged cache in bounded memory, without a GPU: calls whose arguments meet one another, and what the cache refuses
to give up or to reserve."""

import ctypes

import pytest
import torch

from tests.test_gpu_bounded_paths import CALLS, shape_of
from tests.test_paged_host import block, chunks_by_lengths, lib, plan  # noqa: F401


@pytest.mark.parametrize("offset", [0, 4, -4])
def test_new_lengths_over_the_old_ones_are_refused(lib, offset):
    """Blocks read the lengths while others write the new ones.  (No workspace: nothing is launched either way.)"""
    p = block(weight=4096)
    evict = lambda new: lib.rfsn_paged_evict(ctypes.byref(p), 16, 4, 4, new, None, 0, None)
    assert evict(p.lens + offset) == -1
    assert b"new_lens" in lib.rfsn_last_error(), lib.rfsn_last_error()
    for apart in (8, -8):  # two sequences' lengths further on, or before
        assert evict(p.lens + apart) == -1
        assert b"workspace" in lib.rfsn_last_error(), lib.rfsn_last_error()


def quiet_cache(monkeypatch, batch, calls=None, pages=64, **kw):
    """A cache on the host whose kernels do nothing; attention calls' (lens, table, held) go to ``calls``."""
    from apple_amd import kernels as K
    from apple_amd.paged import RFSNPagedKVCache
    from tests.test_paged_host import config

    def attention(q, pages, table, lens, scale, chosen=None, held=0, weight=None):
        if calls is not None:
            calls.append((q, table.clone(), lens.tolist(), held, weight))
        return q + 1

    monkeypatch.setattr(K, "paged_append", lambda pages, table, lens, k, v, cu=None, weight=None: None)
    monkeypatch.setattr(K, "paged_evict", lambda pages, table, lens, weight, keep, *, first, last: lens.clamp_max(keep))
    monkeypatch.setattr(K, "paged_attention", attention)
    monkeypatch.setattr(K, "page_select", lambda *a: torch.zeros((batch, 2, 2), dtype=torch.int32))
    return RFSNPagedKVCache(config(), batch=batch, pages=pages, page_size=16, device="cpu", weights=True, **kw)


def rows(n):
    return torch.zeros((n, 2, 64), dtype=torch.float16)


def test_tokens_without_weights_are_not_chosen_among(monkeypatch):
    """A prompt's rows have weight 0 until a token attends them: an eviction by it would keep the oldest of them."""
    c = quiet_cache(monkeypatch, 2)
    q = torch.zeros((2, 8, 64))
    c.prefill(0, rows(300), rows(300))
    before = (c.num_tokens[:], c.free_pages, c.table.clone())
    with pytest.raises(ValueError, match="300 newest tokens of sequence 0"):
        c.evict(100)
    c.attention_forward(q, sparse_pages=2)  # adds no weights
    with pytest.raises(ValueError, match="weight"):
        c.evict(100)
    assert (c.num_tokens, c.free_pages) == before[:2] and torch.equal(c.table, before[2])
    c.evict(300)   # nothing to give up
    c.evict(100, 30, 70)  # nothing to choose
    assert c.num_tokens == [100, 0]
    with pytest.raises(ValueError, match="weight"):
        c.evict(80)
    c.attention_forward(q)
    c.evict(80)
    assert c.num_tokens == [80, 0]
    # a chunk of a prompt behind it: its newest `last` are kept whatever they weigh, the others not
    c.prefill(0, rows(65), rows(65))
    with pytest.raises(ValueError, match="65 newest"):
        c.evict(90)
    c.evict(90, last=65)
    assert c.num_tokens == [90, 0]
    # the other sequence has no more than it may keep
    c.append(rows(50), rows(50), [0, 50])
    c.attention_forward(q)
    c.append(rows(40), rows(40), [0, 40])
    c.evict(90, last=10)
    with pytest.raises(ValueError, match="40 newest tokens of sequence 1"):
        c.evict(60, last=30)
    c.release(1)
    c.evict(60, last=30)
    assert c.num_tokens == [60, 0]
    c.append(rows(200), rows(200), [0, 200])
    with pytest.raises(ValueError, match="200 newest tokens of sequence 1"):
        c.evict(80)


def test_tokens_without_weights_after_an_eviction_without_a_choice(monkeypatch):
    """Those kept at either end still count."""
    c = quiet_cache(monkeypatch, 1)
    c.prefill(0, rows(40), rows(40))
    c.attention_forward(torch.zeros((1, 8, 64)))
    c.prefill(0, rows(60), rows(60))
    c.evict(70, 50, 20)  # 10 of the 60 among the first 50, 20 among the last
    with pytest.raises(ValueError, match="30 newest"):
        c.evict(60, 4, 29)
    c.evict(60, 4, 30)
    assert c.num_tokens == [60]


def score_bytes(q, table, page_size):
    return table.shape[0] * table.shape[1] * page_size * q.shape[1] * 4


@pytest.mark.parametrize("lens, most", [
    ([2000] + [10] * 40, None), ([10] * 40 + [2000], None), ([10] * 20 + [1500] + [10] * 20 + [500] + [0] * 9, 5),
    ([500, 10] * 4 + [0, 0, 3], 9), ([100] * 20, 1), ([0, 0, 1], 1), ([16 * 100 // (i + 1) for i in range(30)], 8)])
def test_scores_never_need_more_than_the_pool(monkeypatch, lens, most):
    """A batch under one wide table would need room for its scores by its longest sequence, times the batch."""
    from apple_amd import paged

    calls, batch = [], len(lens)
    c = quiet_cache(monkeypatch, batch, calls, pages=sum(-(-n // 16) for n in lens) + 2)
    c.append(rows(sum(lens)), rows(sum(lens)), lens)
    q = torch.arange(batch * 8 * 64, dtype=torch.float32).view(batch, 8, 64).remainder(512)
    out = c.attention_forward(q)
    assert len(calls) == 1 and torch.equal(out, q + 1)  # 256 MiB are no matter
    del calls[:]
    monkeypatch.setattr(paged, "SCORES_AT_LEAST", 0)
    c._unseen = [n for n in lens]
    out = c.attention_forward(q)
    assert torch.equal(out, q + 1) and out.dtype == q.dtype and c._unseen == [0] * batch
    assert len(calls) <= (most or 4), len(calls)
    assert [n for call in calls for n in call[2]] == lens
    b = 0
    for x, table, n, held, weight in calls:
        assert weight is c.weight and torch.equal(x, q[b:b + len(n)].half())
        assert torch.equal(table, c.table[b:b + len(n), :table.shape[1]])
        assert all(-(-t // 16) <= table.shape[1] for t in n) and held == sum(-(-t // 16) for t in n)
        assert score_bytes(x, table, 16) <= c.pages.k.shape[0] * 16 * 8 * 4
        b += len(n)
    # without weights there are no scores
    del calls[:]
    c.weight = None
    c.attention_forward(q)
    assert len(calls) == 1


def test_a_query_without_heads_is_left_to_the_kernels_check(monkeypatch):
    c = quiet_cache(monkeypatch, 1, calls := [])
    c.append(rows(5), rows(5), [5])
    c.attention_forward(torch.zeros((1, 0, 64)))
    assert calls[0][0].shape == (1, 0, 64)


def test_scores_of_a_long_sequence_among_short_ones(monkeypatch):
    calls = []
    c = quiet_cache(monkeypatch, 64, calls, pages=8700, max_tokens=140000)
    lens = [16 * 4] * 20 + [131072] + [16 * 6] * 43
    c.append(rows(sum(lens)), rows(sum(lens)), lens)
    c.attention_forward(torch.zeros((64, 32, 64)))
    assert [len(n) for _, _, n, _, _ in calls] == [20, 16, 28]
    assert max(score_bytes(q, table, 16) for q, table, *_ in calls) <= 256 << 20  # 1,074 MB in one


@pytest.mark.parametrize("call", CALLS)
def test_calls_take_the_variants_that_they_are_for(plan, call):
    """The GPU tests' calls: which blocks they run in, how rows are loaded, how many chunks there are."""
    c = CALLS[call]
    for kind, code in (("fp16", 0), ("int8", 1), ("e4m3", 2), ("e2m1", 4)):
        for dim in c["dims"]:
            pages, width = shape_of(call, kind, dim)
            kw = dict(type=code, batch=len(c["lens"]), pages=pages, table_width=width, table_stride=width, page_size=c["size"],
                      kv_heads=c["kv"], head_dim=dim, head_stride=c["size"] * dim, page_stride=c["kv"] * c["size"] * dim)
            if code:
                kw.update(k_scale=4096, v_scale=4096)
            cut = plan(c["kv"] * c["group"], **kw)
            assert max(c["lens"]) <= width * c["size"]
            assert (cut["wide"], cut["once"], cut["per_seq"] != 1) == (c["wide"], c["once"], c["cut"]), (kind, dim, cut)
            if call == "full" and code == 4:  # three and more chunks of two sequences, by one of the ways to cut at least
                assert len(set(cut["one_over"])) == (3 if dim == 128 else 1), cut
            if not c["cut"]:
                continue
            sizes = list(chunks_by_lengths(cut, c["lens"]))
            if call == "many_tiles":
                assert min(longest for _, longest in sizes) > 32 * 4 * 32  # tiles of 32 positions, 4 waves, 32 at once
            if call.startswith("many_chunks"):
                for one_over in cut["one_over"]:
                    size = max(cut["chunk"], -(-int(sum(c["lens"]) * one_over + 0.98) // 128) * 128)
                    assert -(-max(c["lens"]) // size) > 64
    if call.startswith("second_round"):
        heads = c["kv"] * len(c["lens"])
        assert max(c["lens"]) > 1024 * -(-4096 // heads)


@pytest.mark.parametrize("dim", [64, 128])
def test_a_list_of_pages_takes_chunks_of_many_tiles(plan, dim):
    cut = plan(4096, count=330, type=4, k_scale=4096, v_scale=4096, batch=1, table_width=1250, table_stride=1250, pages=1253,
               page_size=64, kv_heads=1, head_dim=dim, head_stride=64 * dim, page_stride=64 * dim)
    assert not cut["wide"] and cut["per_seq"] > 1 and cut["chunk"] > 32 * 4 * 32
