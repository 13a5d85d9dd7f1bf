"""Prompts of different lengths, padded to one: what the padding holds does not matter."""
import pytest
import torch

from multitokenatention_triton_b200 import PagedKVCache
from test_gpu_generation import module, step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("kind", ["mta", "conv"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
@torch.no_grad()
def test_padding_behind_a_prompt(kind, dtype, poison):
    H, kv, D, counts = 8, 4, 64, [70, 3, 33, 64, 65]
    m, _ = module(H, (6, 11), (3, 3), dtype, kind=kind)
    x = [torch.randn(len(counts), h, 70, D, device=DEV).to(dtype) for h in (H, kv, kv)]
    nxt = [torch.randn(len(counts), h, 1, D, device=DEV).to(dtype) for h in (H, kv, kv)]
    outs = []
    for fill in (0.0, poison):
        for b, n in enumerate(counts):
            for t in x:
                t[b, :, n:] = fill
        given = [t.clone() for t in x]
        cache = PagedKVCache(H, D, 12, 5, 128, m.query_history, n_kv_heads=kv, dtype=dtype)
        slots = [cache.add() for _ in counts]
        out = step(m, kind, *x, cache, cache.extend(slots, counts))
        outs.append([out[b, :, :n].clone() for b, n in enumerate(counts)] + [step(m, kind, *nxt, cache, cache.extend(slots, 1))])
        for t, g in zip(x, given):
            assert torch.equal(t.nan_to_num(7.0), g.nan_to_num(7.0))             # the caller's tensors are as they were
        cache.check()
    for a, b in zip(*outs):
        assert bool(torch.isfinite(b).all())
        assert torch.equal(a, b)
