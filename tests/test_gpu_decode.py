"""One new token over a paged cache (mta_decode_fwd, conv_attn_decode_fwd) against float64, at the sizes where tiles, pages, runs of
tiles and head groups end, with NaN wherever no token is."""
import pytest
import torch

from multitokenatention_triton_b200 import _lib, ops
from paged_ref import Pool, assert_near, mta_weights, token64

pytestmark = pytest.mark.gpu
DEV = "cuda"

# (H, kv heads, D, page, conv kernel, second conv kernel, lengths)
CASES = [
    (16, 16, 128, 64, (6, 11), (3, 3), [301, 1, 64, 65, 0, 7, 63, 128]),
    (8, 8, 64, 16, (3, 5), (3, 3), [2, 15, 16, 17, 31, 33, 200]),
    (4, 4, 128, 64, (6, 11), (3, 3), [2500]),                       # one sequence over many runs
    (3, 3, 40, 32, (2, 3), (1, 1), [5, 100, 32]),                   # heads that are no multiple of four, odd head dimension
    (8, 2, 128, 64, (6, 11), (3, 3), [90, 257]),                    # four query heads a key-value head
    (12, 6, 80, 128, (4, 7), (2, 3), [130, 12]),
    (1, 1, 8, 16, (1, 1), (1, 1), [1, 40]),                         # plain attention of one head
    (5, 1, 64, 64, (7, 7), (7, 7), [3, 70]),                        # five heads on one
    (2, 2, 64, 64, (11, 15), (11, 15), [9, 150]),                   # 21 query rows
    (2, 2, 32, 64, (2, 33), (2, 33), [20, 80]),                     # the widest kernels
    (2, 2, 32, 64, (16, 2), (17, 4), [20, 80]),                     # even key taps, 32 query rows
    (64, 64, 64, 64, (3, 3), (3, 3), [70]),
    (128, 128, 32, 16, (2, 3), (2, 3), [40, 17]),                   # heads taken in parts
]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(pool, got, order, weights, scale, mta):
    for row, s in enumerate(order):
        if pool.lens[s] == 0:
            assert bool((got[row] == 0).all()), f"row {row}: an empty sequence gets zeros"
            continue
        ref, bound = token64(pool.q[s], pool.k[s], pool.v[s], weights[0], scale, *(weights[1:] if mta else ()))
        assert_near(got[row, :, 0], ref, bound, f"row {row} of {pool.lens[s]} tokens")


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"h{c[0]}kv{c[1]}d{c[2]}p{c[3]}k{c[4][0]}x{c[4][1]}k{c[5][0]}x{c[5][1]}")
def test_mta_token_against_float64(case, dtype):
    H, kv, D, page, kernel, kernel2, lens = case
    rows = kernel[0] + kernel2[0] - 1
    pool = Pool(lens, H, kv, D, page, rows + (page == 64), dtype, DEV, seed=len(lens))
    w = mta_weights(H, kernel, kernel2, dtype, DEV)
    got = ops.mta_decode_fwd(*pool.tensors(), *w, max(lens))
    assert got.shape == (len(lens), H, 1, D) and got.dtype == dtype
    check(pool, got, range(len(lens)), w, D ** -0.5, True)
    _lib.cache_status()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"h{c[0]}kv{c[1]}d{c[2]}p{c[3]}k{c[4][0]}x{c[4][1]}")
def test_conv_attention_token_against_float64(case, dtype):
    H, kv, D, page, kernel, _, lens = case
    pool = Pool(lens, H, kv, D, page, kernel[0] + (page == 16), dtype, DEV, seed=len(lens))
    w = mta_weights(H, kernel, (1, 1), dtype, DEV)
    scale = 0.7 * D ** -0.5
    got = ops.conv_attn_decode_fwd(*pool.tensors(), w[0], scale, max(lens))
    check(pool, got, range(len(lens)), w, scale, False)
    _lib.cache_status()


@pytest.mark.parametrize("D", [136, 200, 256])
@pytest.mark.parametrize("kv", [1, 2, 4])
def test_wide_heads(D, kv):
    lens = [37, 100]
    pool = Pool(lens, 4, kv, D, 32, 8, torch.bfloat16, DEV)
    w = mta_weights(4, (6, 11), (3, 3), torch.bfloat16, DEV)
    check(pool, ops.mta_decode_fwd(*pool.tensors(), *w, 100), range(2), w, D ** -0.5, True)
    check(pool, ops.conv_attn_decode_fwd(*pool.tensors(), w[0], None, 100), range(2), w, D ** -0.5, False)


@pytest.mark.parametrize("kv", [16, 4])
def test_long_and_ragged_batches(kv):
    """Runs that begin in one sequence and end in another, sequences of many runs, a batch of many short ones."""
    for lens in ([6000, 10, 3000, 500], [40 + 3 * i for i in range(70)]):
        pool = Pool(lens, 16, kv, 64, 128, 8, torch.bfloat16, DEV, seed=kv)
        w = mta_weights(16, (6, 11), (3, 3), torch.bfloat16, DEV)
        check(pool, ops.mta_decode_fwd(*pool.tensors(), *w, max(lens)), range(len(lens)), w, 0.125, True)
        check(pool, ops.conv_attn_decode_fwd(*pool.tensors(), w[0], 0.125, max(lens)), range(len(lens)), w, 0.125, False)


def test_slots_in_any_order_repeated_and_a_larger_longest_length():
    lens = [50, 0, 130, 3, 64]
    pool = Pool(lens, 8, 8, 64, 32, 9, torch.float16, DEV)
    w = mta_weights(8, (5, 5), (2, 3), torch.float16, DEV)
    order = [4, 2, 2, 1, 0]
    slots = torch.tensor(order, dtype=torch.int32, device=DEV)
    for longest in (130, pool.table.shape[1] * 32):
        check(pool, ops.mta_decode_fwd(*pool.tensors(), *w, longest, slots=slots), order, w, 0.125, True)
        check(pool, ops.conv_attn_decode_fwd(*pool.tensors(), w[0], 0.125, longest, slots=slots), order, w, 0.125, False)


def test_weights_in_float32_and_of_mixed_types():
    pool = Pool([77, 20], 8, 8, 64, 32, 8, torch.bfloat16, DEV)
    w = mta_weights(8, (6, 11), (3, 3), torch.float32, DEV)
    check(pool, ops.mta_decode_fwd(*pool.tensors(), *w, 77), range(2), w, 0.125, True)
    mixed = [w[0], w[1].bfloat16(), w[2], w[3].bfloat16()]
    check(pool, ops.mta_decode_fwd(*pool.tensors(), *mixed, 77), range(2), mixed, 0.125, True)
    check(pool, ops.conv_attn_decode_fwd(*pool.tensors(), w[0], 0.125, 77), range(2), w, 0.125, False)


@pytest.mark.parametrize("spread", [30.0, 200.0])
def test_sharp_softmax_rows(spread):
    """Logits far apart: the running maximum moves late, early parts of a row fade to nothing."""
    pool = Pool([600], 4, 4, 64, 64, 8, torch.float32, DEV)
    ramp = torch.linspace(-spread, spread, 600, device=DEV)
    pool.k[0][:] = ramp[None, :, None] / 64 ** 0.5
    pool.q[0][:] = 1.0
    for t in range(600):
        pool.k_pages[pool.table[0, t // 64], :, t % 64] = pool.k[0][:, t]
    pool.q_hist.fill_(1.0)
    w = mta_weights(4, (6, 11), (3, 3), torch.float32, DEV)
    check(pool, ops.mta_decode_fwd(*pool.tensors(), *w, 600), range(1), w, 0.125, True)
    check(pool, ops.conv_attn_decode_fwd(*pool.tensors(), w[0], 0.125, 600), range(1), w, 0.125, False)


@pytest.mark.parametrize("kernel,kernel2", [((1, 1), (1, 1)), ((6, 11), (3, 3)), ((2, 33), (2, 33)), ((3, 32), (2, 2))])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_a_sequence_that_is_not_finite_leaves_the_others_alone(kernel, kernel2, poison):
    """Every other sequence of a batch whose runs hold several has keys and values that are no numbers."""
    lens = [20 + 7 * (i % 6) for i in range(90)]
    pool = Pool(lens, 4, 4, 64, 16, 8, torch.bfloat16, DEV)
    for s in range(0, 90, 2):
        pages = pool.table[s, :-(-lens[s] // 16)].long()
        pool.k_pages[pages], pool.v_pages[pages] = poison, poison
    w = mta_weights(4, kernel, kernel2, torch.bfloat16, DEV)
    for mta in (True, False):
        got = ops.mta_decode_fwd(*pool.tensors(), *w, max(lens)) if mta else ops.conv_attn_decode_fwd(*pool.tensors(), w[0], 0.125, max(lens))
        for s in range(1, 90, 2):
            ref, bound = token64(pool.q[s], pool.k[s], pool.v[s], w[0], 0.125, *(w[1:] if mta else ()))
            assert_near(got[s, :, 0], ref, bound, f"row {s} of {lens[s]} tokens")
        assert not bool(torch.isfinite(got[::2]).any())


def test_results_do_not_change_from_call_to_call():
    pool = Pool([900, 411, 64], 16, 16, 128, 64, 8, torch.bfloat16, DEV)
    w = mta_weights(16, (6, 11), (3, 3), torch.bfloat16, DEV)
    a = [ops.mta_decode_fwd(*pool.tensors(), *w, 900) for _ in range(3)] + [ops.conv_attn_decode_fwd(*pool.tensors(), w[0], 0.1, 900) for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2]) and torch.equal(a[3], a[4]) and torch.equal(a[3], a[5])


def test_out_and_workspace_of_the_caller():
    pool = Pool([200, 31], 8, 8, 64, 32, 8, torch.bfloat16, DEV)
    w = mta_weights(8, (6, 11), (3, 3), torch.bfloat16, DEV)
    L = _lib.lib()
    n = L.mta_decode_workspace_bytes(2, 8, 8, 64, 6, 11, 3, 3, 200)
    ws = torch.full((n + 64,), 0xFF, dtype=torch.uint8, device=DEV)                   # NaN in every float of it
    out = torch.empty(2, 8, 1, 64, dtype=torch.bfloat16, device=DEV)
    assert ops.mta_decode_fwd(*pool.tensors(), *w, 200, out=out, workspace=ws[:n]) is out
    check(pool, out, range(2), w, 0.125, True)
    assert bool((ws[n:] == 0xFF).all())
    n = L.mta_conv_attn_decode_workspace_bytes(2, 8, 8, 64, 6, 11, 200)
    ws.fill_(0xFF)
    check(pool, ops.conv_attn_decode_fwd(*pool.tensors(), w[0], 0.125, 200, out=out, workspace=ws[:n]), range(2), w, 0.125, False)
    assert bool((ws[n:] == 0xFF).all())


def test_on_another_stream():
    pool = Pool([333, 80], 8, 8, 64, 64, 8, torch.bfloat16, DEV)
    w = mta_weights(8, (6, 11), (3, 3), torch.bfloat16, DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops.mta_decode_fwd(*pool.tensors(), *w, 333)
        b = ops.conv_attn_decode_fwd(*pool.tensors(), w[0], 0.125, 333)
    side.synchronize()
    check(pool, a, range(2), w, 0.125, True)
    check(pool, b, range(2), w, 0.125, False)


def test_calls_at_once_on_two_streams():
    pools = [Pool([700, 90], 8, 8, 64, 64, 8, torch.bfloat16, DEV, seed=i) for i in range(2)]
    w = mta_weights(8, (6, 11), (3, 3), torch.bfloat16, DEV)
    alone = [ops.mta_decode_fwd(*p.tensors(), *w, 700) for p in pools] + [ops.conv_attn_decode_fwd(*p.tensors(), w[0], 0.125, 700) for p in pools]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = {}
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i] = ops.mta_decode_fwd(*pools[i].tensors(), *w, 700)
                outs[2 + i] = ops.conv_attn_decode_fwd(*pools[i].tensors(), w[0], 0.125, 700)
    torch.cuda.synchronize()
    for i in range(4):
        assert torch.equal(outs[i], alone[i])


def test_an_append_is_seen_by_the_attention_behind_it():
    """The calls of a step follow one another without a pause: what the append writes is read, over many steps."""
    pool = Pool([64, 17], 8, 8, 64, 64, 8, torch.bfloat16, DEV, spare=4)
    free = [p for p in range(pool.k_pages.shape[0]) if p not in {int(x) for s, n in enumerate(pool.lens) for x in pool.table[s, :-(-n // 64)]}]
    pool.table[0, 1] = free[0]
    w = mta_weights(8, (6, 11), (3, 3), torch.bfloat16, DEV)
    new = torch.randn(40, 3, 2, 8, 1, 64, device=DEV).bfloat16()
    outs = []
    for q, k, v in new:
        pool.lengths += 1
        ops.cache_append(k, v, q, *(pool.tensors()[i] for i in (1, 2, 0, 3, 4)))
        outs.append((ops.mta_decode_fwd(*pool.tensors(), *w, 110), ops.conv_attn_decode_fwd(*pool.tensors(), w[0], 0.125, 110)))
    for s in range(2):
        q, k, v = (torch.cat([old[s], new[:, i, s, :, 0].transpose(0, 1)], 1) for i, old in enumerate((pool.q, pool.k, pool.v)))
        for n in (1, 2, 25, 39, 40):
            have = pool.lens[s] + n
            for kind in (0, 1):
                ref, bound = token64(q[:, :have], k[:, :have], v[:, :have], w[0], 0.125, *(() if kind else w[1:]))
                assert_near(outs[n - 1][kind][s, :, 0], ref, bound, f"slot {s}, {n} tokens on")
    _lib.cache_status()


def test_captured_graphs_follow_lengths_and_tables():
    """Two graphs captured with workspaces of their own serve shorter and longer sequences than those they were captured with."""
    pool = Pool([100, 30], 8, 8, 64, 32, 8, torch.bfloat16, DEV)
    later = Pool([333, 1], 8, 8, 64, 32, 8, torch.bfloat16, DEV, seed=5)
    w = mta_weights(8, (6, 11), (3, 3), torch.bfloat16, DEV)
    pages = max(pool.k_pages.shape[0], later.k_pages.shape[0])
    width = max(pool.table.shape[1], later.table.shape[1])
    buf = [torch.zeros(2, 8, 8, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(pages, 8, 32, 64, dtype=torch.bfloat16, device=DEV),
           torch.zeros(pages, 8, 32, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, width, dtype=torch.int32, device=DEV),
           torch.zeros(2, dtype=torch.int32, device=DEV)]

    def put(p):
        for b, t in zip(buf, p.tensors()):
            b.zero_()
            b[tuple(slice(0, n) for n in t.shape)].copy_(t)

    put(pool)
    ops.mta_decode_fwd(*buf, *w, width * 32), ops.conv_attn_decode_fwd(*buf, w[0], 0.125, width * 32)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for call in (lambda: ops.mta_decode_fwd(*buf, *w, width * 32), lambda: ops.conv_attn_decode_fwd(*buf, w[0], 0.125, width * 32)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for p in (pool, later, pool):
        put(p)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        check(p, outs[0], range(2), w, 0.125, True)
        check(p, outs[1], range(2), w, 0.125, False)


def test_what_is_out_of_range_is_not_touched_and_reported():
    """Pages, slots and lengths out of range: the other rows are right, the status says so once."""
    lens = [100, 40, 70]
    w = mta_weights(8, (6, 11), (3, 3), torch.bfloat16, DEV)
    for plant in ("page", "negative page", "length", "negative length", "slot"):
        pool = Pool(lens, 8, 8, 64, 32, 8, torch.bfloat16, DEV)
        slots = torch.arange(3, dtype=torch.int32, device=DEV)
        if plant == "page":
            pool.table[1, 0] = pool.k_pages.shape[0]
        elif plant == "negative page":
            pool.table[1, 0] = -1
        elif plant == "length":
            pool.lengths[1] = 101
        elif plant == "negative length":
            pool.lengths[1] = -5
        else:
            slots[1] = 3
        for mta in (True, False):
            _lib.cache_status()
            got = ops.mta_decode_fwd(*pool.tensors(), *w, 100, slots=slots) if mta else ops.conv_attn_decode_fwd(*pool.tensors(), w[0], 0.125, 100, slots=slots)
            with pytest.raises(_lib.MTALibraryError, match="out of range"):
                _lib.cache_status()
            _lib.cache_status()
            if "page" not in plant:
                assert bool((got[1] == 0).all())
            for row in (0, 2):
                ref, bound = token64(pool.q[row], pool.k[row], pool.v[row], w[0], 0.125, *(w[1:] if mta else ()))
                assert_near(got[row, :, 0], ref, bound, plant)
