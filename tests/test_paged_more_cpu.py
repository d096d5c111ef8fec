"""The paged cache's host side: what a caller could break or overlap (no GPU)."""
import ctypes

import pytest
import torch

from sta import _lib as L
from sta import paged
from test_paged_cpu import cache_args, decode_args, evict_args, refused


@pytest.mark.parametrize("name", ["k", "v", "table", "lens", "weights", "device"])
def test_the_tensors_of_a_cache_cannot_be_exchanged(name):
    """The addresses are taken once: another tensor under the same name would go unread, and the
    one that the kernels go on using would be freed."""
    cache = paged.PagedCache.__new__(paged.PagedCache)
    cache._tensors = tuple(torch.zeros(i + 1) for i in range(5)) + (torch.device("cpu"),)
    with pytest.raises(AttributeError):
        setattr(cache, name, torch.zeros(9))
    assert cache.k.numel() == 1 and cache.lens.numel() == 4 and cache.device.type == "cpu"
