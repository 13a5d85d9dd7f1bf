"""What becomes of tokens that PagedKVCache.extend() has reserved, on the CPU: the copies and writes that its kernels make stood in for."""
import gc
import random
import weakref

import pytest
import torch

from multitokenatention_triton_b200 import CacheFullError, PagedKVCache, ops
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


def test_tokens_that_were_never_written_are_not_passed_over(plain_calls):
    """A refused or forgotten append leaves tokens that the attention would read: the next append raises, and truncate() takes them back."""
    c = small()
    a, b = c.add(), c.add()
    c.extend([a], 5)                                        # forgotten: nothing was written at all
    with pytest.raises(MTALibraryError, match="truncate"):
        put(c, c.extend([a], 1), [[9]])
    c.truncate(a, 0)
    put(c, c.extend([a, b], [3, 20]), [[1, 2, 3], list(range(20))])
    gone = c.extend([a, b], [2, 1])                         # refused, say
    batch = c.extend([a, b], 1)
    for layer in (0, 1):
        with pytest.raises(MTALibraryError, match="truncate"):
            put(c, batch, [[9], [9]], layers=[layer])
    c.truncate(a, 3), c.truncate(b, 20)
    for stale in (gone, batch):
        with pytest.raises(MTALibraryError, match="stale"):
            put(c, stale, [[9], [9]])
    put(c, c.extend([a, b], [1, 2]), [[4], [20, 21]])
    for layer in (0, 1):
        assert read(c, a, layer) == [1, 2, 3, 4] and read(c, b, layer) == list(range(22))


def test_a_layer_that_was_left_out(plain_calls):
    c = small()
    a = c.add()
    put(c, c.extend([a], 4), [[1, 2, 3, 4]])
    put(c, c.extend([a], 1), [[5]], layers=[0])             # refused in the second layer
    batch = c.extend([a], 1)
    put(c, batch, [[6]], layers=[0])
    with pytest.raises(MTALibraryError, match="layer 1 was given 4"):
        put(c, batch, [[6]], layers=[1])
    with pytest.raises(MTALibraryError, match="queries"):
        c.truncate(a, 4)                                    # layer 0 has dropped a query that token 4 looks back on
    c.truncate(a, 0)
    put(c, c.extend([a], 6), [[1, 2, 3, 4, 5, 6]])
    assert read(c, a, 0) == read(c, a, 1) == [1, 2, 3, 4, 5, 6]


def test_a_fork_of_unwritten_tokens(plain_calls):
    c = small()
    a = c.add()
    put(c, c.extend([a], 20), [list(range(20))])
    c.extend([a], 1)
    f, = c.fork(a)
    for s in (a, f):
        with pytest.raises(MTALibraryError, match="truncate"):
            put(c, c.extend([s], 1), [[9]])
        c.truncate(s, 20)
    put(c, c.extend([f, a], [1, 2]), [[30], [40, 41]])
    for layer in (0, 1):
        assert read(c, f, layer) == list(range(20)) + [30] and read(c, a, layer) == list(range(20)) + [40, 41]


def test_truncate_gives_pages_back(plain_calls):
    c = small()
    a = c.add()
    put(c, c.extend([a], 20), [list(range(20))])
    f, = c.fork(a)
    c.extend([a], 40)
    assert c.free_pages == 7
    c.truncate(a, 33)
    assert c.free_pages == 8 and c.length(a) == 33 == int(c.lengths[a])
    c.truncate(a, 20)
    assert c.free_pages == 9                                # the copy of the shared page stays
    put(c, c.extend([a], 1), [[50]])
    assert read(c, a) == list(range(20)) + [50] and read(c, f) == list(range(20))
    c.truncate(f, 0)
    assert c.free_pages == 10 and int(c.lengths[f]) == 0 and read(c, a) == list(range(20)) + [50]
    c.truncate(f, 0)
    put(c, c.extend([f], 2), [[7, 8]])
    assert read(c, f) == [7, 8]
    c.free(a), c.free(f)
    assert c.free_pages == 12 and c._refs == [0] * 12


def test_truncate_goes_back_as_far_as_the_queries_reach(plain_calls):
    c = small()                                             # keeps three queries
    a = c.add()
    put(c, c.extend([a], 3), [[1, 2, 3]])
    c.truncate(a, 1)                                        # nothing dropped yet
    put(c, c.extend([a], 2), [[12, 13]])
    assert read(c, a) == [1, 12, 13]
    put(c, c.extend([a], 2), [[14, 15]])
    c.truncate(a, 5)                                        # nothing to do
    c.truncate(a, 4)
    for bad in (3, 1, 5, -1):
        with pytest.raises(MTALibraryError, match="truncate"):
            c.truncate(a, bad)
    put(c, c.extend([a], 1), [[25]])
    assert read(c, a) == [1, 12, 13, 14, 25]
    with pytest.raises(MTALibraryError, match="no sequence"):
        c.truncate(3, 0)


def test_what_others_write_is_not_judged(plain_calls, monkeypatch):
    """Replays of a captured append and writes through the tensors that layer() hands out are not seen: the appends behind them are taken, and
    truncate() takes it that all that was reserved was written."""
    c = small()
    a, b = c.add(), c.add()
    put(c, c.extend([a, b], 4), [[1, 2, 3, 4]] * 2)
    monkeypatch.setattr(PagedKVCache, "_capturing", lambda self: True)
    put(c, c.extend([a], 1), [[5]])
    monkeypatch.undo()
    with pytest.MonkeyPatch.context() as m:
        m.setattr(ops, "cache_append", lambda *args, **kw: None)
        for _ in range(3):
            c.extend([a], 1)                                # replays write these
        batch = c.extend([a], 1)
        c.append(batch, torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1, 8))
        with pytest.raises(MTALibraryError, match="queries"):
            c.truncate(a, 7)
        c.truncate(a, 8)
        with pytest.raises(MTALibraryError, match="queries"):
            c.truncate(a, 7)
        c.free(a)
        assert c.add() == a                                 # the graph's replays write the slot's next sequence too
        c.extend([a], 3)
        x = torch.zeros(1, 2, 1, 8)
        c.append(c.extend([a], 1), x, x, x)
        c.extend([b], 1)
        with pytest.raises(MTALibraryError, match="layer 0 was given 4"):
            c.append(c.extend([b], 1), x, x, x)
        c.layer(0)
        batch = c.extend([b], 1)
        c.append(batch, x, x, x)
        with pytest.raises(MTALibraryError, match="layer 1 was given 4"):
            c.append(batch, x, x, x, 1)


def test_padding_is_cleared():
    c = small()
    slots = [c.add() for _ in range(3)]
    x = [torch.full((3, h, 7, 8), float("nan")) for h in (2, 1)]
    for b, n in enumerate((3, 7, 1)):
        for t in x:
            t[b, :, :n] = 1.0 + b
    batch = c.extend(slots, [3, 7, 1])
    for given, got in zip(x, batch.without_padding(*x)):
        assert got.shape == given.shape
        for b, n in enumerate(batch.counts):
            assert bool((got[b, :, :n] == 1.0 + b).all()) and bool((got[b, :, n:] == 0).all())
        assert bool(given[0, :, 3:].isnan().all())          # the caller's are as they were
    full = c.extend([slots[0]], 7)
    assert full.without_padding(x[0])[0] is x[0]


def test_a_batch_of_another_cache(plain_calls):
    """Two caches whose sequences have gone through the same calls."""
    c, d = small(), small()
    for x in (c, d):
        x.add()
        put(x, x.extend([0], 4), [[1, 2, 3, 4]])
    of_c, of_d = c.extend([0], 1), d.extend([0], 1)
    with pytest.raises(MTALibraryError, match="another cache"):
        put(d, of_c, [[5]])
    put(d, of_d, [[5]])
    big = small(sequences=9)
    late = [big.add() for _ in range(9)][-1]
    with pytest.raises(MTALibraryError, match="another cache"):
        put(c, big.extend([late], 1), [[5]])
    put(c, of_c, [[6]])
    assert read(c, 0) == [1, 2, 3, 4, 6] and read(d, 0) == [1, 2, 3, 4, 5]


@pytest.mark.parametrize("seed", range(12))
def test_random_life_with_truncations(plain_calls, seed):
    """Extensions that are written, forgotten or written in one layer only, truncations, forks, ends and compactions, against lists of tokens:
    what is left is what was written, and the queries that the next token looks back on are there."""
    r = random.Random(seed)
    c = small(pages=24, sequences=6, longest=80)
    held, token = {}, 0

    def lived(s):
        for layer in (0, 1):
            n = c.length(s)
            assert n == int(c.lengths[s]) == len(held[s])
            for pos, t in enumerate(held[s]):
                assert float(c.k_pages[layer, int(c.table[s, pos // 16]), 0, pos % 16, 0]) == t
            for pos in range(max(0, n - c.history + 1), n):
                assert float(c.q_hist[layer, s, pos % c.history, 0, 0]) == held[s][pos]

    for _ in range(200):
        op = r.choice(["add", "extend", "extend", "extend", "refused", "truncate", "truncate", "fork", "free", "compact"])
        slots = r.sample(sorted(held), r.randint(1, len(held))) if held else []
        s = slots[0] if slots else None
        try:
            if op == "add":
                held[c.add()] = []
            elif op in ("extend", "refused") and held:
                counts = [r.choice([1, 1, 2, 17]) for _ in slots]
                batch = c.extend(slots, counts)
                new = [list(range(token + 1 + sum(counts[:i]), token + 1 + sum(counts[:i + 1]))) for i in range(len(counts))]
                token += sum(counts)
                if op == "extend":
                    put(c, batch, new)
                    for x, t in zip(slots, new):
                        held[x] = held[x] + t
                else:
                    half = r.random() < 0.5
                    if half:
                        put(c, batch, new, layers=[0])
                    if r.random() < 0.3:
                        c.compact()
                    for x, n in zip(slots, counts):
                        with pytest.raises(MTALibraryError):
                            put(c, c.extend([x], 1), [[0]], layers=[1])
                        try:
                            c.truncate(x, len(held[x]))
                        except MTALibraryError:
                            assert half and n > 1 and len(held[x]) > 0      # layer 0 dropped queries
                            c.truncate(x, 0)
                            held[x] = []
            elif op == "truncate" and held:
                n = r.choice([0, len(held[s]), max(0, len(held[s]) - 1), r.randint(0, len(held[s]))])
                try:
                    c.truncate(s, n)
                    held[s] = held[s][:n]
                except MTALibraryError:
                    assert 0 < n < len(held[s]) and c._high[s] + len(held[s]) > c.history
            elif op == "fork" and held:
                for new in c.fork(s, r.randint(0, 2)):
                    held[new] = list(held[s])
            elif op == "free" and held:
                c.free(s)
                del held[s]
            elif op == "compact":
                c.compact()
        except CacheFullError:
            for x in held:
                if c.length(x) != len(held[x]):             # extend() of the step that was to be refused found no page
                    c.truncate(x, len(held[x])) if len(held[x]) in (0, c.length(x) - 1) else c.truncate(x, 0)
                    held[x] = held[x] if c.length(x) else []
        for x in held:
            lived(x)
        counts = [0] * 24
        for pages in c._pages:
            for p in pages or ():
                counts[p] += 1
        assert counts == c._refs and sorted(c._free_pages) == [p for p in range(24) if counts[p] == 0]
