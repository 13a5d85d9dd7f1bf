"""Caches whose pages, rows or queries no call over a cache would take are refused when they are made."""
import pytest
import torch

from multitokenatention_triton_b200 import PagedKVCache
from multitokenatention_triton_b200._lib import MTALibraryError


@pytest.mark.parametrize("args", [dict(page_size=1 << 17), dict(page_size=1 << 16, max_length=(1 << 30) + 1), dict(max_length=(1 << 30) + 1),
                                  dict(max_length=1 << 40), dict(page_size=1 << 16, n_heads=1024, n_kv_heads=1024), dict(n_heads=1024, n_kv_heads=1, history=1 << 16),
                                  dict(n_layers=16385)])
def test_refusals(args):
    # on the meta device: nothing is allocated
    a = dict(n_heads=4, head_dim=8, num_pages=2, max_sequences=1, max_length=9, history=2, dtype=torch.float32, device="meta")
    PagedKVCache(**a)
    with pytest.raises(MTALibraryError, match="PagedKVCache"):
        PagedKVCache(**(a | args))


def test_the_largest():
    a = dict(n_heads=4, head_dim=8, num_pages=2, max_sequences=1, history=2, dtype=torch.float32, device="meta")
    assert PagedKVCache(max_length=1 << 30, page_size=1 << 16, **a).table.shape == (1, 1 << 14)
    assert PagedKVCache(max_length=(1 << 30) - 20, **a).table.shape == (1, 1 << 24)
