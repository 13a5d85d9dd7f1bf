"""A step that forward_cached refuses, and how a sequence goes on behind it."""
import pytest
import torch

from multitokenatention_triton_b200 import PagedKVCache
from multitokenatention_triton_b200._lib import MTALibraryError
from paged_ref import assert_near, token64
from test_gpu_generation import module, step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("kind", ["mta", "conv"])
@torch.no_grad()
def test_a_sequence_goes_on_behind_a_refused_step(kind):
    H, D, dtype = 4, 64, torch.bfloat16
    m, w = module(H, (6, 11), (3, 3), dtype, kind=kind)
    cache = PagedKVCache(H, D, 8, 1, 96, m.query_history, page_size=16, dtype=dtype)
    cache.k_pages.fill_(float("nan")), cache.v_pages.fill_(float("nan"))
    s = cache.add()
    x = [torch.randn(1, H, 33, D, device=DEV).to(dtype) for _ in range(3)]

    def some(a, b):
        return [t[:, :, a:b] for t in x]

    step(m, kind, *some(0, 30), cache, cache.extend([s], 30))
    with pytest.raises(NotImplementedError, match="prompt"):
        step(m, kind, *some(30, 32), cache, cache.extend([s], 2))
    with pytest.raises(MTALibraryError, match="truncate"):
        step(m, kind, *some(30, 31), cache, cache.extend([s], 1))
    cache.truncate(s, 30)
    for n in (31, 32, 33):
        out = step(m, kind, *some(n - 1, n), cache, cache.extend([s], 1))
        ref, bound = token64(*(t[0, :, :n] for t in x), w[0], D ** -0.5, *w[1:])
        assert_near(out[0, :, 0], ref, bound, f"{n} tokens")
    cache.truncate(s, 32)                                           # the newest token once more, with other keys and values
    other = [torch.randn_like(t[:, :, :1]) for t in x]
    out = step(m, kind, *other, cache, cache.extend([s], 1))
    ref, bound = token64(*(torch.cat([t[0, :, :32], o[0]], 1) for t, o in zip(x, other)), w[0], D ** -0.5, *w[1:])
    assert_near(out[0, :, 0], ref, bound, "another token 32")
    cache.check()


@torch.no_grad()
def test_a_prefix_that_the_program_wrote_itself():
    """Keys, values and queries put into the tensors of layer(): the tokens behind them are taken, and read them."""
    H, D, dtype = 4, 64, torch.bfloat16
    m, w = module(H, (6, 11), (3, 3), dtype)
    source, cache = (PagedKVCache(H, D, 8, 1, 96, m.query_history, page_size=16, dtype=dtype) for _ in range(2))
    x = [torch.randn(1, H, 31, D, device=DEV).to(dtype) for _ in range(3)]
    for c in (source, cache):
        assert c.add() == 0
    step(m, "mta", *(t[:, :, :30] for t in x), source, source.extend([0], 30))
    cache.extend([0], 30)
    for mine, theirs in zip(cache.layer(0)[:3], source.layer(0)[:3]):
        mine.copy_(theirs)
    out = step(m, "mta", *(t[:, :, 30:] for t in x), cache, cache.extend([0], 1))
    ref, bound = token64(*(t[0] for t in x), w[0], D ** -0.5, *w[1:])
    assert_near(out[0, :, 0], ref, bound)
