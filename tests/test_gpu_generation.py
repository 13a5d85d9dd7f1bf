"""The cache, the append and the attention together, as a program that generates uses them: a prompt, single tokens, forks, ends, a
compaction, a captured step - against the modules' forward over the whole sequence and against float64."""
import types

import pytest
import torch

from multitokenatention_triton_b200 import MTAAttentionTriton, PagedKVCache, TritonConvAttention, _lib
from paged_ref import assert_near, mta_weights, token64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def module(H, kernel, kernel2, dtype, seed=0, pad_key="both", kind="mta"):
    w = mta_weights(H, kernel, kernel2, dtype, DEV, seed)
    if kind == "conv":
        m = TritonConvAttention(H, kernel, causal=True).to(DEV, dtype)
        with torch.no_grad():
            m.weight.copy_(w[0])
        return m, (w[0],)
    cfg = types.SimpleNamespace(use_mta=True, query_kernel_size=kernel[0], key_kernel_size=kernel[1], after_sm_query_kernel_size=kernel2[0],
                                after_sm_key_kernel_size=kernel2[1], pre_sm_linear_head=True, post_sm_linear_head=True, pad_key=pad_key,
                                init_method="identity", dim=H * 64)
    m = MTAAttentionTriton(H, cfg, dropout=0.1, causal=True).to(DEV, dtype).eval()
    with torch.no_grad():
        for p, t in zip((m.mta_conv_triton.weight, m.wpsm_triton.weight, m.mta_conv_after_sm_triton.weight, m.wposm_triton.weight), w):
            p.copy_(t)
        return m, (m.mta_conv_triton.effective_weight().clone(), w[1], m.mta_conv_after_sm_triton.effective_weight().clone(), w[3])


def step(m, kind, q, k, v, cache, batch, **more):
    """(B,H,T,D) whatever the module's own layout is."""
    if kind == "conv":
        return m.forward_cached(q, k, v, cache, batch, **more)[0]
    return m.forward_cached(q, k, v, cache, batch, **more).transpose(1, 2)


@pytest.mark.parametrize("kind", ["mta", "conv"])
@pytest.mark.parametrize("H,kv,D,page,dtype", [(16, 16, 128, 64, torch.bfloat16), (8, 2, 64, 16, torch.float16), (4, 4, 32, 32, torch.float32)])
@torch.no_grad()
def test_a_conversation(kind, H, kv, D, page, dtype):
    m, w = module(H, (6, 11), (3, 3), dtype, kind=kind)
    cache = PagedKVCache(H, D, 40 * 64 // page, 6, 400, m.query_history, page_size=page, n_kv_heads=kv, n_layers=2, dtype=dtype)
    g = torch.Generator(device=DEV).manual_seed(3)
    scale = D ** -0.5
    said = {}                                                       # slot -> [q, k, v] of all its tokens, (heads, n, D)

    def draw(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    def tokens(slots, counts):
        """New tokens of some sequences through both layers (the second has its own keys); checks the newest of each."""
        T = max(counts)
        batch = cache.extend(slots, counts)
        per_layer = [(draw(len(slots), H, T, D), draw(len(slots), kv, T, D), draw(len(slots), kv, T, D)) for _ in range(2)]
        outs = [step(m, kind, *x, cache, batch, layer=i) for i, x in enumerate(per_layer)]
        for row, (s, n) in enumerate(zip(slots, counts)):
            for i, x in enumerate(per_layer):
                old = said.get((s, i))
                new = [t[row, :, :n] for t in x]
                said[s, i] = new if old is None else [torch.cat([a, b], 1) for a, b in zip(old, new)]
                ref, bound = token64(*said[s, i], w[0], scale, *w[1:])
                got = outs[i][row, :, n - 1]
                if T == 1:
                    assert_near(got, ref, bound, f"slot {s} layer {i}")
                else:                                               # the whole-sequence forward rounds between its stages
                    err = float((got.double() - ref).norm() / ref.norm())
                    assert err < {torch.float32: 1e-5, torch.float16: 6e-3, torch.bfloat16: 4e-2}[dtype], err
        return outs

    a, b, c = cache.add(), cache.add(), cache.add()
    tokens([a, b, c], [70, 3, 33])                                  # prompts, padded on the right
    for _ in range(3):
        tokens([c, a], [1, 1])
    f1, f2 = cache.fork(a, 2)
    for f in (f1, f2):
        for i in range(2):
            said[f, i] = said[a, i]
    for _ in range(2):
        tokens([f1, a, b, f2], [1, 1, 1, 1])
    cache.free(a)
    cache.free(c)
    d = cache.add()
    for key in [k for k in said if k[0] == d]:
        del said[key]
    tokens([d], [1])                                                # a prompt of one token
    tokens([f2, f1, d], [1, 1, 1])
    used = cache.compact()
    assert used == cache.num_pages - cache.free_pages
    for _ in range(page + 2):                                       # over a page's end
        tokens([b, d, f2], [1, 1, 1])
    tokens([f1], [1])
    cache.check()
    _lib.device_status()


@pytest.mark.parametrize("pad_key", ["left", "right"])
@torch.no_grad()
def test_pad_key_and_even_kernels(pad_key):
    for kernel, kernel2, pad in (((4, 6), (3, 3), pad_key), ((3, 4), (2, 6), "both")):
        m, w = module(4, kernel, kernel2, torch.bfloat16, pad_key=pad)
        cache = PagedKVCache(4, 64, 4, 1, 100, m.query_history, dtype=torch.bfloat16)
        s = cache.add()
        q, k, v = (torch.randn(1, 4, 50, 64, device=DEV).bfloat16() for _ in range(3))
        out = m.forward_cached(q[:, :, :49], k[:, :, :49], v[:, :, :49], cache, cache.extend([s], 49))
        assert out.shape == (1, 49, 4, 64)
        got = m.forward_cached(q[:, :, 49:], k[:, :, 49:], v[:, :, 49:], cache, cache.extend([s], 1))
        ref, bound = token64(q[0], k[0], v[0], w[0], 0.125, *w[1:])
        assert_near(got[0, 0], ref, bound)


@torch.no_grad()
def test_a_captured_step_generates_as_the_plain_one():
    """One graph of append and attention, replayed over a page's end while the host extends the sequences between replays."""
    m, _ = module(8, (6, 11), (3, 3), torch.bfloat16)
    tokens = [torch.randn(3, 2, 8, 1, 64, device=DEV).bfloat16() for _ in range(40)]
    start = [torch.randn(2, 8, 20, 64, device=DEV).bfloat16() for _ in range(3)]
    results = []
    for captured in (False, True):
        cache = PagedKVCache(8, 64, 12, 2, 128, m.query_history, page_size=32, dtype=torch.bfloat16)
        slots = [cache.add(), cache.add()]
        m.forward_cached(*start, cache, cache.extend(slots, 20))
        x = [t.clone() for t in tokens[0]]
        outs, graph = [], None
        for t in tokens:
            batch = cache.extend(slots, 1)
            for buf, new in zip(x, t):
                buf.copy_(new)
            if not captured:
                outs.append(m.forward_cached(*x, cache, batch))
            elif graph is None:
                outs.append(m.forward_cached(*x, cache, batch, max_length=cache.max_length))    # the first of its kind on the device
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    static = m.forward_cached(*x, cache, batch, max_length=cache.max_length)
                keep = batch                                         # its slot ids are what the graph reads
            else:
                graph.replay()
                outs.append(static.clone())
        cache.check()
        results.append((outs, [cache.k_pages.clone(), cache.lengths.clone()]))
    assert keep.slots == tuple(slots)
    for a, b in zip(results[0][0], results[1][0]):
        # another longest length cuts the work otherwise: float32 sums in another order, rounded once
        assert float((a.double() - b.double()).abs().max()) <= 2.0 ** -7 * float(a.double().abs().max())
    assert torch.equal(results[0][1][1], results[1][1][1])
