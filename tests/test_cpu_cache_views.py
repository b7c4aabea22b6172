"""Views that page copies may and may not address."""
import pytest
import torch

from omni_npu_b200 import ops


@pytest.mark.parametrize("t", [
    torch.zeros(1, 8, 16, 32).expand(4, 8, 16, 32),                        # one page under four names
    torch.zeros(4, 1, 16, 32).expand(4, 8, 16, 32),
    torch.zeros(1, 16, 32).expand(4, 16, 32),
    torch.zeros(4096).as_strided((4, 2, 4, 8), (32, 32, 8, 1)),            # a page's second head is the next one's first
    torch.zeros(4096).as_strided((4, 4, 8), (16, 8, 1)),
])
def test_overlapping_pages_are_refused(t):
    with pytest.raises(ValueError, match="overlap"):
        ops.CacheBlocks([t])


@pytest.mark.parametrize("t", [
    torch.zeros(4, 2, 16, 32),
    torch.zeros(2, 4, 16, 32).transpose(0, 1),                             # heads outermost
    torch.zeros(4, 2, 3, 16, 32)[:, 1],                                    # keys and values of a page side by side
    torch.zeros(3, 4, 16, 32)[1],
    torch.zeros(1, 8, 16, 32).expand(1, 8, 16, 32),
    torch.zeros(8, 16, 32)[::2],
])
def test_other_views_are_taken(t):
    g = torch.Generator().manual_seed(1)
    t.copy_(torch.randn(t.shape, generator=g))
    want = t.clone()
    cache = ops.CacheBlocks([t])
    if t.shape[0] > 2:
        ops.copy_blocks(cache, [(0, 2, 5)])
        want[2, ..., :5, :] = want[0, ..., :5, :]
    assert torch.equal(t, want)
