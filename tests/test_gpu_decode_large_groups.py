"""MTA decoding with more query heads on a key-value head than have room for their scores at once."""
import pytest
import torch

from multitokenatention_triton_b200 import _lib, ops
from paged_ref import Pool, assert_near, mta_weights, token64

pytestmark = pytest.mark.gpu
DEV = "cuda"

# (H, kv heads, D, conv kernel, second conv kernel)
SHAPES = [
    (64, 1, 64, (6, 11), (3, 3)),
    (128, 8, 32, (6, 11), (3, 3)),
    (128, 1, 16, (6, 11), (3, 3)),
    (63, 1, 32, (6, 11), (3, 3)),                                   # parts of an odd number of heads, taken in pairs
    (127, 1, 16, (4, 5), (2, 3)),                                   # parts of one head
    (96, 3, 32, (6, 11), (3, 3)),
    (32, 2, 64, (11, 15), (11, 15)),
    (64, 2, 128, (6, 11), (3, 3)),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H,kv,D,kernel,kernel2", SHAPES)
def test_parts_of_a_group(H, kv, D, kernel, kernel2, dtype):
    lens = [70, 17, 0, 300, 1]
    pool = Pool(lens, H, kv, D, 32, kernel[0] + kernel2[0] - 1, dtype, DEV)
    w = mta_weights(H, kernel, kernel2, dtype, DEV)
    got = ops.mta_decode_fwd(*pool.tensors(), *w, 300)
    assert bool((got[2] == 0).all())
    for s, n in enumerate(lens):
        if n:
            ref, bound = token64(pool.q[s], pool.k[s], pool.v[s], w[0], D ** -0.5, *w[1:])
            assert_near(got[s, :, 0], ref, bound, f"{n} tokens")
    _lib.cache_status()


def test_large_groups_in_a_long_batch():
    """Runs that begin in one sequence and end in another, with parts of a group."""
    lens = [33 + 11 * i for i in range(40)]
    pool = Pool(lens, 64, 1, 64, 64, 8, torch.bfloat16, DEV)
    w = mta_weights(64, (6, 11), (3, 3), torch.bfloat16, DEV)
    got = ops.mta_decode_fwd(*pool.tensors(), *w, max(lens))
    for s, n in enumerate(lens):
        ref, bound = token64(pool.q[s], pool.k[s], pool.v[s], w[0], 0.125, *w[1:])
        assert_near(got[s, :, 0], ref, bound, f"{n} tokens")
