"""A paged cache in bounded memory on the GPU, where other calls than test_gpu_bounded.py's lead: in-place results among
a program's gradients, and the kernels' variants for large calls, against 64 bits."""

import pytest
import torch

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
