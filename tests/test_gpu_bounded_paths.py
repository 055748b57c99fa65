"""A paged cache in bounded memory on the GPU, where other calls than test_gpu_bounded.py's lead: in-place results among
a program's gradients, and the kernels' variants for large calls, against 64 bits."""

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
