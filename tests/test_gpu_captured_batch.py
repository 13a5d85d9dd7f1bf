"""A captured decoding step whose batch the caller does not keep, as a loop that binds it anew for every token does."""
import gc

import pytest
import torch

from multitokenatention_triton_b200 import PagedKVCache
from paged_ref import assert_near, token64
from test_gpu_generation import module, step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("kind", ["mta", "conv"])
@torch.no_grad()
def test_replays_after_the_batch_was_bound_anew(kind):
    H, D, dtype = 4, 64, torch.bfloat16
    m, w = module(H, (6, 11), (3, 3), dtype, kind=kind)
    cache = PagedKVCache(H, D, 24, 4, 96, m.query_history, page_size=16, dtype=dtype)
    other, *slots = [cache.add() for _ in range(4)]
    slots = [slots[2], slots[0]]
    said = {s: [torch.randn(H, 20, D, device=DEV).to(dtype) for _ in range(3)] for s in (other, *slots)}
    step(m, kind, *(torch.stack([said[s][i] for s in said]) for i in range(3)), cache, cache.extend(list(said), 20))
    x = [torch.empty(2, H, 1, D, device=DEV, dtype=dtype) for _ in range(3)]

    def speak():
        batch = cache.extend(slots, 1)
        for i, t in enumerate(x):
            t.normal_()
            for row, s in enumerate(slots):
                said[s][i] = torch.cat([said[s][i], t[row]], 1)
        return batch

    step(m, kind, *x, cache, speak(), max_length=cache.max_length)
    batch = speak()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step(m, kind, *x, cache, batch, max_length=cache.max_length)
    graph.replay()
    litter = []
    for _ in range(20):
        batch = speak()
        gc.collect()
        litter += [torch.zeros(n, dtype=torch.int32, device=DEV) for n in (1, 2, 4, 8, 128)]     # slot 0 and counts of 0 where ids are freed
        before = cache.k_pages.clone(), cache.q_hist[0, other].clone()
        graph.replay()
        for row, s in enumerate(slots):
            ref, bound = token64(*said[s], w[0], D ** -0.5, *w[1:])
            assert_near(static[row, :, 0], ref, bound, f"slot {s} after {cache.length(s)} tokens")
        pages = cache.table[other, :2].long()
        # bit by bit: places that hold no token may be NaN
        for now, then in ((cache.k_pages[0, pages], before[0][0, pages]), (cache.q_hist[0, other], before[1])):
            assert torch.equal(now.view(torch.int16), then.view(torch.int16))
    cache.check()
