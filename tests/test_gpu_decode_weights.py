"""The product of one new token's weights with the values: how many bits the weights have, for any number of heads that share
keys; values that are infinite."""
import pytest
import torch

from multitokenatention_triton_b200 import ops
from paged_ref import HALF_STEP, Pool, assert_near, mta_weights, token64

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H,kv", [(4, 4), (4, 2), (4, 1), (8, 1)])
@pytest.mark.parametrize("mta", [True, False])
def test_weights_keep_the_bits_of_float32(mta, H, kv, dtype):
    """Plain attention over three keys with logits -a, -a - d and 0 and values c, -c and 0: the result is the difference of two weights that
    agree in twelve bits, so that an error of the weights shows.

    Bound.  A logit is at most 1.2 in magnitude; its sum, its scaled tap and the conversion to base 2 are off by 2^-22 of it at most, the
    exponential by 2^-22, its sums by less: 2^-20.5 of a weight, 2^-19.5 of it for the difference of two.  On top of that comes
    the result's own rounding.  Weights of sixteen bits would be off by 2^-17 each."""
    B, D, page, d = 64, 64, 16, 2.0 ** -12
    a = (0.2 + 0.6 * torch.arange(B, device=DEV) / B).bfloat16()
    pool = Pool([3] * B, H, kv, D, page, 1, dtype, DEV)
    c = torch.linspace(0.5, 2.0, D, device=DEV).bfloat16().to(dtype)
    at = pool.table[:, 0].long()
    pool.q_hist.zero_()
    pool.q_hist[..., :2] = 1.0
    pool.k_pages[at, :, :3] = 0.0
    pool.k_pages[at, :, 0, 0] = pool.k_pages[at, :, 1, 0] = -a[:, None].to(dtype)
    pool.k_pages[at, :, 1, 1] = -d
    pool.v_pages[at, :, 0], pool.v_pages[at, :, 1], pool.v_pages[at, :, 2] = c, -c, 0.0
    s = torch.linspace(0.7, 1.15, H, device=DEV)
    one = torch.ones(H, 1, 1, device=DEV)
    if mta:
        eye = torch.eye(H, device=DEV)
        got = ops.mta_decode_fwd(*pool.tensors(), (8.0 * s)[:, None, None].contiguous(), eye, one, eye, 3)
    else:
        got = ops.conv_attn_decode_fwd(*pool.tensors(), s[:, None, None].contiguous(), 1.0, 3)
    z = a.double()[:, None] * s.double()
    p0, p1 = torch.exp(-z), torch.exp(-z - d * s.double())
    l = (1.0 + p0 + p1)[..., None]
    ref = (p0 - p1)[..., None] / l * c.double()
    allowed = p0[..., None] / l * c.double() * 2.0 ** -19.5 + HALF_STEP[dtype] * ref.abs()
    off = (got[:, :, 0].double() - ref).abs()
    assert bool((off <= allowed).all()), f"{int((off > allowed).sum())} of {off.numel()} off by more than allowed, the worst {float((off / allowed).max()):.1f} times"


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H,kv", [(4, 4), (4, 2), (4, 1), (8, 1)])
@pytest.mark.parametrize("mta", [True, False])
def test_infinite_values(mta, H, kv, dtype):
    """An infinite value times a positive weight is that infinity, whatever numbers the weight is split into; two of both signs make NaN; every
    other element is as if there were none.  Lengths of one run and of many."""
    lens, D = [40, 900, 17], 64
    pool = Pool(lens, H, kv, D, 32, 8, dtype, DEV)
    for s, n in enumerate(lens):
        for key, e, x in ((3, 5, 1.0), (n - 1, 6, -1.0), (n // 2, 40, 1.0), (0, 63, 1.0), (n - 2, 63, -1.0)):
            pool.v[s][:, key, e] = x * float("inf")
            pool.v_pages[pool.table[s, key // 32], :, key % 32, e] = x * float("inf")
    w1, _, w2, _ = mta_weights(H, (6, 11), (3, 3), dtype, DEV)
    eye = torch.eye(H, device=DEV, dtype=dtype)
    w = (w1, eye, w2.abs(), eye) if mta else (w1,)
    got = ops.mta_decode_fwd(*pool.tensors(), *w, 900) if mta else ops.conv_attn_decode_fwd(*pool.tensors(), w1, 0.125, 900)
    wild = torch.zeros(D, dtype=torch.bool, device=DEV)
    wild[[5, 6, 40, 63]] = True
    for s in range(len(lens)):
        ref, bound = token64(pool.q[s], pool.k[s], pool.v[s], w1, 0.125, *w[1:])
        row = got[s, :, 0]
        assert_near(row[:, ~wild], ref[:, ~wild], bound[:, ~wild], f"row {s}")
        assert bool((row[:, 5] == float("inf")).all() and (row[:, 6] == -float("inf")).all() and (row[:, 40] == float("inf")).all()), row[:, wild]
        assert bool(row[:, 63].isnan().all())
