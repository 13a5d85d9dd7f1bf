"""Sizes that a decoding call would refuse: the workspace sizes say so, and forward_cached refuses the prompt, with nothing written."""
import types

import pytest
import torch

from multitokenatention_triton_b200 import MTAAttentionTriton, PagedKVCache, TritonConvAttention, _lib, ops
from multitokenatention_triton_b200._lib import MTALibraryError


def module(H, kernel, kernel2):
    cfg = types.SimpleNamespace(use_mta=True, query_kernel_size=kernel[0], key_kernel_size=kernel[1], after_sm_query_kernel_size=kernel2[0],
                                after_sm_key_kernel_size=kernel2[1], pre_sm_linear_head=True, post_sm_linear_head=True, pad_key="both",
                                init_method="identity", dim=H * 64)
    return MTAAttentionTriton(H, cfg, dropout=0.0, causal=True).eval()


def test_workspace_sizes_of_refused_shapes_are_zero():
    L = _lib.lib()

    def mta(B=1, H=4, kv=4, D=64, cq=6, ck=11, cq2=3, ck2=3, longest=64):
        return L.mta_decode_workspace_bytes(B, H, kv, D, cq, ck, cq2, ck2, longest)

    def conv(B=1, H=4, kv=4, D=64, cq=6, ck=11, longest=64):
        return L.mta_conv_attn_decode_workspace_bytes(B, H, kv, D, cq, ck, longest)

    assert mta() > 0 and conv() > 0 and mta(B=1024) > 0 and conv(B=1024) > 0 and mta(B=0) > 0 and conv(B=0) > 0
    for bad in (dict(B=-1), dict(B=1025), dict(H=0), dict(kv=3), dict(kv=0), dict(D=4), dict(cq=0), dict(cq=33), dict(ck=0), dict(ck=34), dict(longest=-1),
                dict(B=1024, longest=1 << 25)):
        for size in (mta, conv):
            assert size(**bad) == 0, (size, bad)
            assert L.mta_last_error(), bad
    for bad in (dict(H=129, kv=129), dict(cq2=0), dict(cq2=28), dict(ck2=34), dict(cq=2 ** 31 - 1, cq2=2 ** 31 - 1)):
        assert mta(**bad) == 0 and L.mta_last_error(), bad


@pytest.mark.parametrize("T", [5, 1])
@pytest.mark.parametrize("kernel,kernel2,why", [((11, 33), (12, 33), "shared memory"), ((3, 34), (3, 3), "key taps"), ((3, 3), (3, 35), "key taps"), ((20, 3), (14, 3), "queries")])
@torch.no_grad()
def test_mta_refuses_a_prompt_whose_tokens_it_would_refuse(kernel, kernel2, why, T, monkeypatch):
    m = module(64, kernel, kernel2)
    c = PagedKVCache(64, 8, 4, 1, 32, 40, page_size=16, dtype=torch.float32, device="cpu")
    s = c.add()
    x = torch.zeros(1, 64, T, 8)
    for name in ("cache_append", "mta_fused_fwd", "mta_decode_fwd"):
        monkeypatch.setattr(ops, name, lambda *a, **k: pytest.fail("reached"))
    batch = c.extend([s], T)
    for _ in range(2):                                              # the second time from the sizes that are remembered
        with pytest.raises(MTALibraryError, match=why):
            m.forward_cached(x, x, x, c, batch)
    c.truncate(s, 0)
    assert c.length(s) == 0 and c.free_pages == 4


@pytest.mark.parametrize("T", [5, 1])
@torch.no_grad()
def test_conv_attention_refuses_a_prompt_whose_tokens_it_would_refuse(T, monkeypatch):
    c = PagedKVCache(4, 8, 4, 1, 32, 6, page_size=16, dtype=torch.float32, device="cpu")
    s = c.add()
    x = torch.zeros(1, 4, T, 8)
    for name in ("cache_append", "conv_attn_fwd", "conv_attn_decode_fwd"):
        monkeypatch.setattr(ops, name, lambda *a, **k: pytest.fail("reached"))
    batch = c.extend([s], T)
    with pytest.raises(MTALibraryError, match="key taps"):
        TritonConvAttention(4, (3, 35)).forward_cached(x, x, x, c, batch)
    with pytest.raises(MTALibraryError, match="look back on 7 queries"):
        TritonConvAttention(4, (7, 3)).forward_cached(x, x, x, c, batch)
    with pytest.raises(MTALibraryError, match="8 heads"):
        TritonConvAttention(8, (3, 3)).forward_cached(x, x, x, c, batch)


@torch.no_grad()
def test_a_prompt_is_written_only_once_its_attention_has_run(monkeypatch):
    """A refusal of the whole-sequence forward (an even number of key taps, say) leaves the cache as extend() left it."""
    c = PagedKVCache(4, 8, 4, 2, 32, 6, page_size=16, dtype=torch.float32, device="cpu")
    s = c.add()
    x = torch.zeros(1, 4, 5, 8)
    calls = []

    def refuse(*a, **k):
        calls.append("attention")
        raise MTALibraryError("refused")

    monkeypatch.setattr(ops, "conv_attn_fwd", refuse)
    monkeypatch.setattr(ops, "cache_append", lambda *a, **k: calls.append("append"))
    batch = c.extend([s], 5)
    with pytest.raises(MTALibraryError, match="refused"):
        TritonConvAttention(4, (3, 4)).forward_cached(x, x, x, c, batch)
    assert calls == ["attention"]
    monkeypatch.setattr(ops, "conv_attn_fwd", lambda *a, **k: calls.append("attention"))
    TritonConvAttention(4, (3, 4)).forward_cached(x, x, x, c, batch)            # the batch is good still
    assert calls == ["attention", "attention", "append"]
    old = c.extend([s], 1)
    c.extend([s], 1)
    with pytest.raises(MTALibraryError, match="stale"):
        TritonConvAttention(4, (3, 3)).forward_cached(x[:, :, :1], x[:, :, :1], x[:, :, :1], c, old)
    assert len(calls) == 3
    # a prompt of more rows than one decoding call takes
    many = PagedKVCache(4, 8, 1100, 1100, 16, 6, page_size=16, dtype=torch.float32, device="cpu")
    y = torch.zeros(1100, 4, 2, 8)
    TritonConvAttention(4, (3, 3)).forward_cached(y, y, y, many, many.extend([many.add() for _ in range(1100)], 2))
    assert len(calls) == 5


@pytest.mark.parametrize("H,kv,kernel,kernel2,most", [(64, 1, (6, 11), (3, 3), 256), (128, 8, (6, 11), (3, 3), 128), (128, 128, (6, 11), (3, 3), 128),
                                                      (32, 2, (11, 15), (11, 15), 256), (127, 1, (6, 11), (3, 3), 128), (48, 3, (11, 15), (3, 3), 256)])
def test_groups_of_any_size_fit(H, kv, kernel, kernel2, most):
    """What several heads that share keys need is what as many heads with keys of their own need."""
    L = _lib.lib()
    for D in (64, most):
        for B in (1, 64):
            assert L.mta_decode_workspace_bytes(B, H, kv, D, *kernel, *kernel2, 100) == L.mta_decode_workspace_bytes(B, H, H, D, *kernel, *kernel2, 100) > 0
