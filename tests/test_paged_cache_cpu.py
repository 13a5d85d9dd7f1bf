"""The paged cache's bookkeeping on the CPU (the copies that its kernels make stood in for), and what the cache calls refuse before
they touch a device."""
import ctypes
import random
import types

import pytest
import torch

from multitokenatention_triton_b200 import CacheFullError, MTAAttentionTriton, PagedKVCache, TritonConvAttention, _lib, ops
from multitokenatention_triton_b200._lib import MTALibraryError


@pytest.fixture
def plain_copies(monkeypatch):
    def copy(k, v, src, dst, q=None, slot_src=None, slot_dst=None):
        src, dst = src.long(), dst.long()
        assert len(set(dst.tolist())) == len(dst) and not set(dst.tolist()) & set(src.tolist())
        k[:, dst], v[:, dst] = k[:, src].clone(), v[:, src].clone()
        q[:, slot_dst.long()] = q[:, slot_src.long()].clone()
    monkeypatch.setattr(ops, "cache_copy", copy)


def small(pages=12, sequences=4, longest=96, layers=2):
    c = PagedKVCache(2, 8, pages, sequences, longest, 3, page_size=16, n_layers=layers, dtype=torch.float32, device="cpu")
    c.k_pages.zero_(), c.v_pages.zero_(), c.q_hist.zero_()
    return c


def write(c, batch, tokens):
    """What append writes, with the token's number as every value."""
    for s, n, total, t in zip(batch.slots, batch.counts, batch.lengths, tokens):
        for i in range(n):
            pos = total - n + i
            p = int(c.table[s, pos // c.page_size])
            c.k_pages[:, p, :, pos % c.page_size] = t[i]
            c.v_pages[:, p, :, pos % c.page_size] = -t[i]
            c.q_hist[:, s, pos % c.history] = t[i]


def read(c, s):
    n = int(c.lengths[s])
    assert n == c.length(s)
    out = []
    for pos in range(n):
        p = int(c.table[s, pos // c.page_size])
        k, v = c.k_pages[:, p, :, pos % c.page_size], c.v_pages[:, p, :, pos % c.page_size]
        assert bool((k == k.flatten()[0]).all()) and torch.equal(v, -k)
        out.append(int(k.flatten()[0]))
    for pos in range(max(0, n - c.history), n):
        assert bool((c.q_hist[:, s, pos % c.history] == out[pos]).all())
    return out


def test_extend_hands_out_pages_in_order_and_keeps_the_mirrors():
    c = small()
    a, b = c.add(), c.add()
    assert (a, b) == (0, 1) and c.free_pages == 12 and c.free_slots == 2
    x = c.extend([b, a], [17, 3])
    assert x.slots == (1, 0) and x.counts == (17, 3) and x.lengths == (17, 3) and x.max_length == 17 and x.from_empty
    assert x.slot_ids.tolist() == [1, 0] and x.count_ids.tolist() == [17, 3]
    assert c.lengths.tolist() == [3, 17, 0, 0] and c.table[1, :2].tolist() == [0, 1] and c.table[0, 0] == 2 and c.free_pages == 9
    y = c.extend([a], 13)
    assert c.free_pages == 9 and c.length(a) == 16 and not y.from_empty
    c.extend([a], 1)
    assert c.free_pages == 8 and c.table[0, :2].tolist() == [2, 3]


def test_a_full_cache_changes_nothing():
    c = small(pages=4)
    a, b = c.add(), c.add()
    c.extend([a, b], [20, 10])
    before = (c.lengths.clone(), c.table.clone(), c.free_pages)
    with pytest.raises(CacheFullError):
        c.extend([a, b], [20, 20])
    with pytest.raises(CacheFullError):
        c.extend([a], 77)                                   # longer than the longest
    assert torch.equal(c.lengths, before[0]) and torch.equal(c.table, before[1]) and c.free_pages == before[2] and c.length(a) == 20
    c.add(), c.add()
    with pytest.raises(CacheFullError):
        c.add()
    with pytest.raises(CacheFullError):
        c.fork(a)


@pytest.mark.parametrize("bad", [lambda c: c.extend([0, 0], 1), lambda c: c.extend([0], 0), lambda c: c.extend([0], [1, 2]), lambda c: c.extend([3], 1),
                                 lambda c: c.extend([-1], 1), lambda c: c.free(2), lambda c: c.fork(9), lambda c: c.fork(0, -1), lambda c: c.length(1),
                                 lambda c: c.layer(2), lambda c: c.layer(-1)])
def test_refusals_of_the_bookkeeping(bad):
    c = small()
    c.add()
    with pytest.raises(MTALibraryError):
        bad(c)


@pytest.mark.parametrize("args", [dict(page_size=24), dict(page_size=8), dict(n_kv_heads=3), dict(head_dim=12), dict(head_dim=136), dict(dtype=torch.float64),
                                  dict(history=0), dict(n_layers=0)])
def test_refusals_of_the_constructor(args):
    a = dict(n_heads=4, head_dim=8, num_pages=2, max_sequences=1, max_length=9, history=2, dtype=torch.float32, device="cpu")
    with pytest.raises(MTALibraryError):
        PagedKVCache(**(a | args))


def test_forks_share_pages_until_one_writes(plain_copies):
    c = small()
    a = c.add()
    write(c, c.extend([a], 20), [list(range(1, 21))])
    b, d = c.fork(a, 2)
    assert c.free_pages == 10 and read(c, b) == read(c, d) == read(c, a) == list(range(1, 21))
    write(c, c.extend([a, b, d], [1, 2, 13]), [[100], [200, 201], list(range(300, 313))])
    assert c.free_pages == 7                                # two copies of the shared page, one page more for d
    assert read(c, a) == list(range(1, 21)) + [100]
    assert read(c, b) == list(range(1, 21)) + [200, 201]
    assert read(c, d) == list(range(1, 21)) + list(range(300, 313))
    c.free(a)
    assert c.free_pages == 8 and int(c.lengths[a]) == 0     # the first page is still shared by two
    c.free(b), c.free(d)
    assert c.free_pages == 12 and c.free_slots == 4


def test_a_batch_is_stale_after_its_sequences_change(plain_copies):
    c = small()
    a, b = c.add(), c.add()
    x, y = c.extend([a], 5), c.extend([b], 5)
    c.check_batch(x), c.check_batch(y)                      # other sequences' batches do not matter
    c.extend([a], 1)
    c.check_batch(y)
    with pytest.raises(MTALibraryError, match="stale"):
        c.check_batch(x)
    c.free(b)
    with pytest.raises(MTALibraryError, match="stale"):
        c.append(y, None, None, None)
    b2 = c.add()
    assert b2 == b
    with pytest.raises(MTALibraryError, match="stale"):
        c.check_batch(y)


@pytest.mark.parametrize("seed", range(8))
def test_random_life_of_a_cache(plain_copies, seed):
    """Adds, extensions, forks, ends and compactions in any order, against lists of tokens."""
    r = random.Random(seed)
    c = small(pages=20, sequences=6, longest=80)
    held, token = {}, 0
    for _ in range(150):
        op = r.choice(["add", "extend", "extend", "extend", "fork", "free", "compact"])
        try:
            if op == "add":
                held[c.add()] = []
            elif op == "extend" and held:
                slots = r.sample(sorted(held), r.randint(1, len(held)))
                counts = [r.randint(1, 20) for _ in slots]
                batch = c.extend(slots, counts)
                new = []
                for s, n in zip(slots, counts):
                    new.append(list(range(token + 1, token + n + 1)))
                    token += n
                    held[s] = held[s] + new[-1]
                write(c, batch, new)
            elif op == "fork" and held:
                s = r.choice(sorted(held))
                for new in c.fork(s, r.randint(0, 2)):
                    held[new] = list(held[s])
            elif op == "free" and held:
                s = r.choice(sorted(held))
                c.free(s)
                del held[s]
            elif op == "compact":
                used = c.compact()
                assert all(p < used for pages in c._pages if pages for p in pages) and used == 20 - c.free_pages
        except CacheFullError:
            pass
        for s, tokens in held.items():
            assert read(c, s) == tokens
        counts = [0] * 20
        for pages in c._pages:
            for p in pages or ():
                counts[p] += 1
        assert counts == c._refs and sorted(c._free_pages) == [p for p in range(20) if counts[p] == 0]


def test_longest_length_of_a_call():
    c = small()
    a = c.add()
    batch = c.extend([a], 20)
    assert c.longest(batch, None) == 20 and c.longest(batch, 20) == 20 and c.longest(batch, 96) == 96
    for bad in (19, 97, -1):
        with pytest.raises(MTALibraryError, match="max_length"):
            c.longest(batch, bad)


def test_empty_problems_and_bad_arguments_of_the_c_calls():
    L = _lib.lib()
    z, one = ctypes.c_void_p(0), ctypes.c_void_p(16)
    strides = (ctypes.c_longlong * 9)(*[64] * 9)

    def append(B=1, T=1, slots=2, width=4, pages=8, page=16, ring=3, H=4, kv=2, D=16, dtype=1, k=one, strides=strides):
        return L.mta_cache_append(k, one, one, strides, z, one, one, one, one, one, z, B, T, slots, width, pages, page, ring, H, kv, D, dtype, z)

    assert append(B=0) == 0 and append(T=0) == 0
    for bad in (dict(T=-1), dict(B=-1), dict(B=3), dict(slots=0), dict(width=0), dict(pages=0), dict(page=24), dict(page=8), dict(ring=0), dict(H=0), dict(kv=0),
                dict(kv=3), dict(D=0), dict(D=20), dict(D=264), dict(D=136, dtype=0), dict(dtype=3), dict(k=z), dict(k=ctypes.c_void_p(24)),
                dict(strides=(ctypes.c_longlong * 9)(*[60] * 9)), dict(width=1 << 20, page=65536), dict(width=1 << 15, page=65536)):
        assert append(**bad) == 1, bad
        assert L.mta_last_error()

    def mta(B=1, ws=1 << 30, cq=3, ck=5, cq2=3, ck2=3, longest=64, ring=8, H=4, kv=4, D=16, dtype=1, wd=1, o=one, work=one, slots=2):
        return L.mta_decode_fwd(one, one, one, one, one, z, one, one, one, one, o, work, ws, B, slots, 4, 8, 16, ring, H, kv, D, cq, ck, cq2, ck2, longest, dtype, wd, z)

    def conv(B=1, ws=1 << 30, cq=3, ck=5, longest=64, ring=8, H=4, kv=4, D=16, dtype=1, wd=1, o=one, work=one, slots=2):
        return L.mta_conv_attn_decode_fwd(one, one, one, one, one, z, one, o, work, ws, B, slots, 4, 8, 16, ring, H, kv, D, cq, ck, longest, 1.0, dtype, wd, z)

    for call in (mta, conv):
        assert call(B=0) == 0
        for bad in (dict(B=3), dict(ws=16), dict(cq=0), dict(ck=0), dict(ck=34), dict(cq=9), dict(cq=33, ring=40), dict(longest=65), dict(longest=-1), dict(kv=3),
                    dict(D=12), dict(dtype=7), dict(wd=7), dict(o=z), dict(work=z), dict(work=ctypes.c_void_p(8)), dict(B=1025, slots=2000)):
            assert call(**bad) == 1, (call, bad)
            assert L.mta_last_error()
    for bad in (dict(cq2=0), dict(ck2=34), dict(cq2=7), dict(H=129, kv=129), dict(H=128, kv=128, D=256, cq=16, ck=33, cq2=17, ck2=33, ring=32)):
        assert mta(**bad) == 1, bad
    assert b"shared memory" in L.mta_last_error()
    assert L.mta_decode_workspace_bytes(1, 128, 128, 256, 16, 33, 17, 33, 64) == 0
    assert L.mta_decode_workspace_bytes(1, 3, 2, 64, 3, 3, 3, 3, 64) == 0 and L.mta_conv_attn_decode_workspace_bytes(1, 3, 2, 64, 3, 3, 64) == 0

    def copy(n=1, page_bytes=64, pages=4, m=0, slot_bytes=0, slots=0, layers=1, k=one, q=z, a=z):
        return L.mta_cache_copy(k, one, one, one, n, page_bytes, pages, q, a, a, m, slot_bytes, slots, layers, z)

    assert copy(n=0) == 0
    for bad in (dict(n=-1), dict(m=-1), dict(page_bytes=0), dict(page_bytes=40), dict(page_bytes=1 << 31), dict(pages=0), dict(layers=0), dict(k=z),
                dict(k=ctypes.c_void_p(8)), dict(m=1, slot_bytes=16, slots=1), dict(m=1, slot_bytes=8, slots=1, q=one, a=one), dict(m=1, slot_bytes=16, q=one, a=one)):
        assert copy(**bad) == 1, bad


def test_ops_refuse_what_does_not_belong_together():
    q, k = torch.zeros(2, 3, 4, 16), torch.zeros(5, 2, 16, 16)
    table, lengths = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    w = torch.zeros(4, 3, 3)
    for args in ((q, k, k, table, lengths), (q, k, k, table.long(), lengths), (q[:1], k, k, table, lengths), (q, k, k[:2], table, lengths),
                 (q, k.half(), k.half(), table, lengths), (q, k, k, table, lengths[:1]), (q[0], k, k, table, lengths), (q, k[..., :8], k[..., :8], table, lengths)):
        with pytest.raises(MTALibraryError):                # the first of them only because it is not on a GPU
            ops.conv_attn_decode_fwd(*args, w, None, 64)
    with pytest.raises(MTALibraryError):
        ops.cache_copy(k, k, lengths, lengths)


def test_modules_refuse_training_and_longer_prompts():
    cfg = types.SimpleNamespace(use_mta=True, query_kernel_size=6, key_kernel_size=11, after_sm_query_kernel_size=3, after_sm_key_kernel_size=3,
                                pre_sm_linear_head=True, post_sm_linear_head=True, pad_key="both", init_method="identity", dim=16)
    m = MTAAttentionTriton(2, cfg, dropout=0.1, causal=True)
    assert m.query_history == 8 and TritonConvAttention(2, (6, 11), causal=True).query_history == 6
    c = small()
    a = c.add()
    c.extend([a], 3)
    batch = c.extend([a], 2)
    x = torch.zeros(1, 2, 2, 8)
    with pytest.raises(NotImplementedError, match="dropout"):
        m.forward_cached(x, x, x, c, batch)
    m.eval()
    with pytest.raises(NotImplementedError, match="no_grad"):
        m.forward_cached(x, x, x, c, batch)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="prompt"):
        m.forward_cached(x, x, x, c, batch)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="prompt"):
        TritonConvAttention(2, (3, 3)).forward_cached(x, x, x, c, batch)
    with pytest.raises(NotImplementedError, match="no_grad"):
        TritonConvAttention(2, (3, 3)).forward_cached(x, x, x, c, batch)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="causal"):
        MTAAttentionTriton(2, cfg, dropout=0.0, causal=False).eval().forward_cached(x, x, x, c, batch)
