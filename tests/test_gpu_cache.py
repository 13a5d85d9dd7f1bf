"""Writes into a paged cache (cache_append, cache_copy): every byte that should change does, no other."""
import pytest
import torch

from multitokenatention_triton_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def fresh(slots, width, pages, H, kv, D, page, ring, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    k, v = (torch.randn(pages, kv, page, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    q = torch.randn(slots, ring, H, D, generator=g, device=DEV).to(dtype)
    table = torch.randperm(pages, generator=g, device=DEV)[:slots * width].reshape(slots, width).int().contiguous()
    return k, v, q, table, torch.zeros(slots, dtype=torch.int32, device=DEV)


def plain_append(k, v, q, k_pages, v_pages, q_hist, table, lengths, slots, counts):
    page, ring = k_pages.shape[2], q_hist.shape[1]
    for b, (s, n) in enumerate(zip(slots, counts)):
        for i in range(n):
            pos = int(lengths[s]) - n + i
            p = int(table[s, pos // page])
            k_pages[p, :, pos % page], v_pages[p, :, pos % page] = k[b, :, i], v[b, :, i]
            if i >= n - ring:
                q_hist[s, pos % ring] = q[b, :, i]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,counts,before", [(1, [1, 1, 1], [0, 37, 63]), (70, [70, 1, 33], [0, 15, 16]), (5, [0, 5, 2], [9, 0, 31]), (130, None, [1, 2, 3])])
@pytest.mark.parametrize("H,kv,D,page,ring", [(16, 16, 128, 64, 8), (6, 2, 40, 16, 3), (3, 3, 8, 32, 21)])
def test_append(H, kv, D, page, ring, T, counts, before, dtype):
    order = [3, 0, 2]
    real = counts or [T] * 3
    k_pages, v_pages, q_hist, table, lengths = fresh(4, 14, 60, H, kv, D, page, ring, dtype)
    for s, n, x in zip(order, real, before):
        lengths[s] = n + x
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(3, kv, T, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    q = torch.randn(3, H, T, D, generator=g, device=DEV).to(dtype)
    want = [t.clone() for t in (k_pages, v_pages, q_hist)]
    plain_append(k, v, q, *want, table.cpu(), lengths.cpu(), order, real)
    ops.cache_append(k, v, q, k_pages, v_pages, q_hist, table, lengths, slots=torch.tensor(order, dtype=torch.int32, device=DEV),
                     counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV))
    for got, ref in zip((k_pages, v_pages, q_hist), want):
        assert torch.equal(got, ref)
    _lib.cache_status()


def test_append_of_strided_unaligned_and_broadcast_inputs():
    H, kv, D, T = 8, 4, 64, 9
    base = torch.randn(2, T, H + 2 * kv, D, device=DEV).bfloat16()                # as one projection of q, k and v gives them
    q, k, v = base.transpose(1, 2).split([H, kv, kv], dim=1)
    odd = torch.randn(2 * kv * T * D + 1, device=DEV).bfloat16()[1:].view(2, kv, T, D)
    wide = torch.randn(2, kv, T, D + 4, device=DEV).bfloat16()[..., 2:-2]
    same = torch.randn(1, 1, T, D, device=DEV).bfloat16().expand(2, kv, T, D)
    flipped = torch.randn(2, kv, D, T, device=DEV).bfloat16().transpose(2, 3)
    for k_, v_ in ((k, v), (odd, v), (wide, same), (same, flipped)):
        pools = fresh(2, 2, 8, H, kv, D, 16, 5, torch.bfloat16)
        pools[4].fill_(T + 3)
        want = [t.clone() for t in pools[:3]]
        plain_append(k_, v_, q, *want, pools[3].cpu(), pools[4].cpu(), [0, 1], [T, T])
        ops.cache_append(k_, v_, q, *pools)
        for got, ref in zip(pools, want):
            assert torch.equal(got, ref)


def test_append_skips_and_reports_what_is_out_of_range():
    for plant in ("page", "count", "negative count", "length", "slot"):
        k_pages, v_pages, q_hist, table, lengths = fresh(3, 2, 8, 4, 4, 32, 16, 4, torch.bfloat16)
        lengths.fill_(20)
        counts, slots = torch.full((2,), 3, dtype=torch.int32, device=DEV), torch.tensor([0, 2], dtype=torch.int32, device=DEV)
        k, v, q = (torch.randn(2, 4, 3, 32, device=DEV).bfloat16() for _ in range(3))
        want = [t.clone() for t in (k_pages, v_pages, q_hist)]
        plain_append(k, v, q, *want, table.cpu(), lengths.cpu(), [0, 2], [3, 0])
        if plant == "page":
            table[2, 1] = 99
        elif plant == "count":
            counts[1] = 4
        elif plant == "negative count":
            counts[1] = -1
        elif plant == "length":
            lengths[2] = 33                                                       # a table row holds 32
        else:
            slots[1] = -1
        ops.cache_append(k, v, q, k_pages, v_pages, q_hist, table, lengths, slots=slots, counts=counts)
        assert torch.equal(k_pages, want[0]) and torch.equal(v_pages, want[1])
        if plant != "page":
            assert torch.equal(q_hist, want[2])
        with pytest.raises(_lib.MTALibraryError, match="out of range"):
            _lib.cache_status()


@pytest.mark.parametrize("layers", [None, 3])
@pytest.mark.parametrize("dtype,H,D,page", [(torch.bfloat16, 16, 128, 64), (torch.float32, 3, 8, 16), (torch.float16, 5, 40, 32)])
def test_copy(layers, dtype, H, D, page):
    lead = () if layers is None else (layers,)
    k, v = (torch.randn(*lead, 20, H, page, D, device=DEV).to(dtype) for _ in range(2))
    q = torch.randn(*lead, 6, 8, H, D, device=DEV).to(dtype)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for src, dst, a, b in (((3, 7, 3, 19), (0, 1, 2, 18), (5,), (0,)), ((4,), (5,), (), ()), ((), (), (1, 1), (2, 3))):
        want = [t.clone() for t in (k, v, q)]
        at = (slice(None),) * len(lead)
        for s, d in zip(src, dst):
            want[0][at + (d,)], want[1][at + (d,)] = k[at + (s,)], v[at + (s,)]
        for s, d in zip(a, b):
            want[2][at + (d,)] = q[at + (s,)]
        ops.cache_copy(k, v, i32(*src), i32(*dst), q, i32(*a), i32(*b))
        for got, ref in zip((k, v, q), want):
            assert torch.equal(got, ref)
    _lib.cache_status()
    want = k.clone()
    ops.cache_copy(k, v, i32(0, 20, -1), i32(20, 1, 2))                           # pairs that name no page are skipped
    assert torch.equal(k, want)
    with pytest.raises(_lib.MTALibraryError, match="out of range"):
        _lib.cache_status()
