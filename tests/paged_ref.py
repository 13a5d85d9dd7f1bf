"""One new token over a paged cache in float64, from the definition, with a bound on what float32 kernels may differ by.

The bound follows the computation: every sum of n products done in float32 is off by at most n * U times the sum of the products'
magnitudes (U = 2^-22: four roundings' worth for each, which covers the alignment inside a tensor core's accumulator), errors of
inputs pass through the linear stages with the weights' magnitudes, and a probability's relative error is at most twice the largest
error of the row's logits plus the roundings of the exponent and of the sum.  With 16-bit values the kernels may multiply them with
weights that are sums of two numbers of that type: the first is off by half a step, the second by half a step of that, 2^-16 in bf16
and 2^-22 in fp16, where a number scaled to 2^15 at most is also off by half of 2^-24, 2^-39 of the largest weight.
"""
import torch

U = 2.0 ** -22
PIECES = {torch.float32: 0.0, torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def conv64(x, w):
    """(H, rows, keys) with (H, cq, ck): rows that have all their taps; keys centred as the library centres them."""
    H, cq, ck = w.shape
    left = (ck - 1) // 2
    x = torch.nn.functional.pad(x, (left, ck - 1 - left))
    n, keys = x.shape[1] - cq + 1, x.shape[2] - ck + 1
    y = torch.zeros(H, n, keys, dtype=torch.float64, device=x.device)
    for i in range(cq):
        for j in range(ck):
            y += w[:, i, j, None, None] * x[:, i:i + n, j:j + keys]
    return y


def token64(q, k, v, w1, scale, W1=None, w2=None, W2=None):
    """The newest token of one sequence: q (H,n,D) all its queries, k, v (kv heads,n,D), the weights; all taken to float64.  Returns
    (out (H,D), bound on the absolute error of a float32 evaluation).  Without W1, w2 and W2 the conv attention."""
    dtype = q.dtype
    q, k, v, w1 = q.double(), k.double(), v.double(), w1.double()
    H, n, D = q.shape
    k, v = (t.repeat_interleave(H // t.shape[0], 0) for t in (k, v))
    cq, ck = w1.shape[1:]
    cq2 = 1 if w2 is None else w2.shape[1]
    R = cq + cq2 - 1
    pos = torch.arange(n - R, n, device=q.device)
    key = torch.arange(n, device=q.device)
    seen = (key[None, :] <= pos[:, None])                                     # a row before the first token sees nothing
    rows = torch.where((pos >= 0)[None, :, None], q[:, pos.clamp(min=0)], torch.zeros((), dtype=torch.float64, device=q.device))
    s = torch.where(seen, rows @ k.transpose(1, 2) * scale, 0.0)
    es = torch.where(seen, rows.abs() @ k.abs().transpose(1, 2) * abs(scale), 0.0) * (D + 2) * U
    c, ec = conv64(s, w1), conv64(es, w1.abs()) + conv64(s.abs(), w1.abs()) * (cq * ck + 1) * U
    if W1 is not None:
        W1, w2, W2 = W1.double(), w2.double(), W2.double()
        ec = torch.tensordot(W1.abs(), ec + c.abs() * (H + 1) * U, dims=1)
        c = torch.tensordot(W1, c, dims=1)
    seen = seen[R - cq2:]
    c = torch.where(seen, c, -torch.inf)
    live = (pos[R - cq2:] >= 0)[None, :, None]
    p = torch.where(live, torch.softmax(c, dim=2), 0.0)
    worst = torch.where(seen, ec + c.abs().nan_to_num(posinf=0.0) * 4 * U, 0.0).amax(dim=2, keepdim=True)
    ep = p * (torch.expm1(2 * worst) + (n + 8) * U)
    if W1 is not None:
        y, ey = conv64(p, w2), conv64(ep, w2.abs()) + conv64(p, w2.abs()) * (w2[0].numel() + 1) * U
        p = torch.tensordot(W2, y, dims=1)
        ep = torch.tensordot(W2.abs(), ey + y.abs() * (H + 1) * U, dims=1)
    ep = ep + p.abs() * PIECES[dtype]
    if dtype == torch.float16:
        ep = ep + 2.0 ** -39 * (1.0 if W1 is None else (W2.abs() @ w2.abs().sum((1, 2)))[:, None, None])
    out = (p @ v)[:, 0]
    return out, (ep @ v.abs() + (p.abs() @ v.abs()) * (n + 8) * U)[:, 0]


def assert_near(got, ref, bound, what=""):
    """got rounds ref once in its type and is within the float32 bound besides."""
    got64 = got.double()
    allowed = bound + HALF_STEP[got.dtype] * (ref.abs() + bound) + torch.finfo(got.dtype).tiny
    off = (got64 - ref).abs()
    assert bool((off <= allowed).all()), f"{what}: off by {float((off - allowed).max()):.3e} more than allowed; worst ratio {float((off / allowed).max()):.2f}"


class Pool:
    """A cache's tensors with pages in random order; whatever holds no token is NaN."""

    def __init__(self, lens, H, kv_heads, D, page, ring, dtype, device, seed=0, spare=3, slots=None, poison=True):
        g = torch.Generator(device=device).manual_seed(seed)
        n = len(lens)
        self.lens, self.page, self.ring = list(lens), page, ring
        need = [-(-x // page) for x in lens]
        pages = sum(need) + spare
        width = max(need + [1]) + 1
        fill = float("nan") if poison else 0.0
        self.k_pages = torch.full((pages, kv_heads, page, D), fill, dtype=dtype, device=device)
        self.v_pages = torch.full_like(self.k_pages, fill)
        self.q_hist = torch.full((n, ring, H, D), fill, dtype=dtype, device=device)
        self.table = torch.zeros(n, width, dtype=torch.int32, device=device)
        self.lengths = torch.tensor(list(lens), dtype=torch.int32, device=device)
        perm = torch.randperm(pages, generator=g, device=device)
        self.q, self.k, self.v = [], [], []
        at = 0
        for s, x in enumerate(lens):
            mine = perm[at:at + need[s]]
            at += need[s]
            self.table[s, :need[s]] = mine.int()
            q, k, v = (torch.randn(h, x, D, generator=g, device=device).to(dtype) for h in (H, kv_heads, kv_heads))
            self.q.append(q), self.k.append(k), self.v.append(v)
            for t in range(x):
                p = mine[t // page]
                self.k_pages[p, :, t % page] = k[:, t]
                self.v_pages[p, :, t % page] = v[:, t]
            for t in range(max(0, x - ring), x):
                self.q_hist[s, t % ring] = q[:, t]

    def tensors(self):
        return self.q_hist, self.k_pages, self.v_pages, self.table, self.lengths


def mta_weights(H, kernel, kernel2, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(1000 + seed)

    def conv(r, s):
        w = torch.randn(H, r, s, generator=g, device=device) * (r * s) ** -0.5
        w[:, r - 1, s // 2] += 1.0
        return w.to(dtype)

    def mix():
        return (torch.eye(H, device=device) + 0.02 ** 0.5 * torch.randn(H, H, generator=g, device=device)).to(dtype)

    return conv(*kernel), mix(), conv(*kernel2), mix()
