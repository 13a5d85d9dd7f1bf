"""Forwards whose conv kernels have an even number of key taps, which run stage by stage, against float64 row by row."""
import types

import pytest
import torch

from multitokenatention_triton_b200 import MTAAttentionTriton
from paged_ref import assert_near, mta_weights, token64

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("kernel,kernel2", [((4, 6), (3, 4)), ((3, 4), (2, 3)), ((6, 11), (1, 2)), ((2, 2), (2, 2))])
@torch.no_grad()
def test_even_key_extents(kernel, kernel2):
    H, D, S = 4, 64, 75
    cfg = types.SimpleNamespace(use_mta=True, query_kernel_size=kernel[0], key_kernel_size=kernel[1], after_sm_query_kernel_size=kernel2[0],
                                after_sm_key_kernel_size=kernel2[1], pre_sm_linear_head=True, post_sm_linear_head=True, pad_key="both",
                                init_method="identity", dim=H * D)
    m = MTAAttentionTriton(H, cfg, dropout=0.0, causal=True).to(DEV).eval()
    w = mta_weights(H, kernel, kernel2, torch.float32, DEV)
    for p, t in zip((m.mta_conv_triton.weight, m.wpsm_triton.weight, m.mta_conv_after_sm_triton.weight, m.wposm_triton.weight), w):
        p.copy_(t)
    q, k, v = (torch.randn(2, H, S, D, device=DEV) for _ in range(3))
    out = m(q, k, v, None, None)
    assert out.shape == (2, S, H, D)
    for b in range(2):
        for n in (1, 2, 3, 7, 31, 64, 75):
            ref, bound = token64(q[b, :, :n], k[b, :, :n], v[b, :, :n], w[0], D ** -0.5, *w[1:])
            assert_near(out[b, n - 1], ref, bound, f"sequence {b}, row {n - 1}")
