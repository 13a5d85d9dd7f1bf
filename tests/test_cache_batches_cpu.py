"""What becomes of tokens that PagedKVCache.extend() has reserved, on the CPU: the copies and writes that its kernels make stood in for."""
import gc
import weakref

import pytest
import torch

from multitokenatention_triton_b200 import PagedKVCache, ops
from multitokenatention_triton_b200._lib import MTALibraryError


@pytest.fixture
def plain_calls(monkeypatch):
    def copy(k, v, src, dst, q=None, slot_src=None, slot_dst=None):
        src, dst = src.long(), dst.long()
        k[:, dst], v[:, dst] = k[:, src].clone(), v[:, src].clone()
        q[:, slot_dst.long()] = q[:, slot_src.long()].clone()

    def append(k, v, q, k_pages, v_pages, q_hist, table, lengths, slots=None, counts=None):
        page, ring = k_pages.shape[2], q_hist.shape[1]
        for b, (s, n) in enumerate(zip(slots.tolist(), counts.tolist())):
            for i in range(n):
                pos = int(lengths[s]) - n + i
                p = int(table[s, pos // page])
                k_pages[p, :, pos % page], v_pages[p, :, pos % page], q_hist[s, pos % ring] = k[b, :, i], v[b, :, i], q[b, :, i]

    monkeypatch.setattr(ops, "cache_copy", copy)
    monkeypatch.setattr(ops, "cache_append", append)


def small(pages=12, sequences=4, longest=96, layers=2):
    c = PagedKVCache(2, 8, pages, sequences, longest, 3, page_size=16, n_layers=layers, dtype=torch.float32, device="cpu")
    for t in (c.k_pages, c.v_pages, c.q_hist):
        t.fill_(float("nan"))                               # what no token was written to
    return c


def put(c, batch, tokens, layers=(0, 1)):
    """Appends tokens[b] (numbers) as the keys, values and queries of the batch's rows."""
    x = torch.zeros(len(tokens), 2, max(batch.counts), 8)
    for b, t in enumerate(tokens):
        x[b, :, :len(t)] = torch.tensor(t, dtype=torch.float32)[None, :, None]
    for layer in layers:
        c.append(batch, x, x, x, layer)


def read(c, s, layer=0):
    n = c.length(s)
    assert int(c.lengths[s]) == n
    out = [float(c.k_pages[layer, int(c.table[s, pos // 16]), 0, pos % 16, 0]) for pos in range(n)]
    for pos in range(max(0, n - c.history), n):
        assert float(c.q_hist[layer, s, pos % c.history, 0, 0]) == out[pos]
    return out


def test_a_fork_makes_the_batches_of_its_sequence_stale(plain_calls):
    c = small()
    a = c.add()
    put(c, c.extend([a], 5), [[1, 2, 3, 4, 5]])
    batch = c.extend([a], 1)
    c.fork(a, 0)                                            # no copy, no change
    c.check_batch(batch)
    c.fork(a)
    with pytest.raises(MTALibraryError, match="stale"):
        put(c, batch, [[6]])


def test_a_fork_between_two_layers_of_a_prompt(plain_calls):
    c = small()
    a = c.add()
    batch = c.extend([a], 3)
    put(c, batch, [[1, 2, 3]], layers=[0])
    c.fork(a)
    with pytest.raises(MTALibraryError, match="stale"):
        put(c, batch, [[1, 2, 3]], layers=[1])


def test_a_captured_batch_is_kept(plain_calls, monkeypatch):
    """A graph reads the ids of the batch that it was captured with: they live as long as the cache, whatever the caller binds anew."""
    c = small()
    a, b = c.add(), c.add()
    put(c, c.extend([a, b], [3, 2]), [[1, 2, 3], [4, 5]])
    alive = []
    for capturing in (False, True):
        monkeypatch.setattr(PagedKVCache, "_capturing", lambda self, on=capturing: on)
        batch = c.extend([b, a], 1)
        put(c, batch, [[6], [7]])
        alive.append((weakref.ref(batch.slot_ids), weakref.ref(batch.count_ids)))
        if capturing:
            assert len(c._captured) == 1                    # two layers, one batch
    monkeypatch.undo()
    batch = c.extend([a, b], 1)                             # binds the name anew
    gc.collect()
    assert alive[0][0]() is None and alive[0][1]() is None
    assert alive[1][0]().tolist() == [b, a] and alive[1][1]().tolist() == [1, 1]
