"""The operators that generate token by token over a paged cache, as cases that can be timed and checked one by one.

  mta     one new token per sequence through the whole MTA module: scores of the last queries against every cached key,
          conv, head mix, softmax, conv, head mix, product with the cached values
  conv    one new token per sequence through the conv attention softmax(scale * conv(Q K^T)) V
  append  new tokens' keys, values and queries written into the cache: one per sequence, or whole prompts
  copy    pages moved inside the cache: the partly filled page of a forked sequence, or the pages of a compaction

A cache is a pool of pages (pages, kv heads, tokens, head dim) for the keys and one for the values, a table of page numbers per
sequence, a length per sequence, and a ring of the last queries per sequence, position p at p % ring.  In its plain form every
operator is written with elementary torch operations in float32; with `own` it is this package's call.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _case(name, op, dtype, batch, heads, length, dim=128, kv_heads=0, page=64, kernel=(6, 11), kernel2=(3, 3), ragged=True):
    c = {"op": op, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads or heads, "length": length, "dim": dim,
         "page": page, "cq": kernel[0], "ck": kernel[1], "cq2": kernel2[0], "ck2": kernel2[1], "ragged": ragged}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user in a short conversation: launches and host time count
        _case("mta_b1_l301_bf16", "mta", "bf16", 1, 16, 301, ragged=False),
        # the small float32 configuration of the parity suite, eight sequences
        _case("mta_b8_l1024_fp32", "mta", "fp32", 8, 8, 1024, dim=64, kernel=(3, 5)),
        # the headline configuration after prompts of different lengths
        _case("mta_b8_l4096_bf16", "mta", "bf16", 8, 16, 4096),
        # the large configuration, a full batch of long contexts
        _case("mta_b16_l8192_h32_bf16", "mta", "bf16", 16, 32, 8192, ragged=False),
        # the conv attention for one user
        _case("conv_b1_l517_fp16", "conv", "fp16", 1, 16, 517, dim=64, ragged=False),
        # the widest published kernel, a batch as it comes
        _case("conv_b32_l4096_fp16", "conv", "fp16", 32, 16, 4096, dim=64, kernel=(11, 15)),
        # one very long document: the work has to be split over its length
        _case("conv_b1_l131072_bf16", "conv", "bf16", 1, 16, 131072, ragged=False),
        # key-value heads shared by four query heads each
        _case("conv_b8_l8192_kv8_bf16", "conv", "bf16", 8, 32, 8192, kv_heads=8),
        # the write of a decoding step
        _case("append_b64_t1_bf16", "append", "bf16", 64, 16, 1, ragged=False),
        # prompts of different lengths, padded on the right
        _case("append_b8_t4096_bf16", "append", "bf16", 8, 16, 4096),
        # eight beams, each forked: one partly filled page apiece
        _case("copy_p8_bf16", "copy", "bf16", 1, 16, 8, ragged=False),
        # a compaction of a pool after many sequences have ended
        _case("copy_p1500_bf16", "copy", "bf16", 1, 16, 1500, ragged=False),
    ]


# The most key and value bytes that a drawn case reads.
LIMIT = 1 << 30


def draw(rng):
    op = rng.choice(["mta", "mta", "mta", "conv", "conv", "append", "copy"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dim = rng.choice([32, 64, 64, 80, 128, 128, 128])
    heads = rng.choice([8, 12, 16, 16, 24, 32])
    kv_heads = heads if rng.random() < 0.6 else heads // rng.choice([2, 4])
    kernel = rng.choice([(2, 3), (3, 5), (4, 7), (5, 5), (6, 11), (6, 11), (7, 7), (11, 15)])
    kernel2 = kernel if rng.random() < 0.2 else rng.choice([(1, 1), (2, 3), (3, 3), (3, 3)])
    page = rng.choice([16, 32, 64, 64, 128])
    token = 2 * kv_heads * dim * SIZE[dtype]
    if op == "copy":
        most = min(2000, LIMIT // (2 * token * page))
        return _case(None, op, dtype, 1, heads, round(most ** rng.random()), dim, kv_heads, page, kernel, kernel2, False)
    if op == "append":
        # float32 of the plain form's work counts for the decoding operators alone; a prompt is at most 4096 tokens long
        length = rng.choice([1, 1, round(4096 ** rng.random())])
        batch = max(1, min(round(64 ** rng.random()), LIMIT // (8 * token * length)))
        return _case(None, op, dtype, batch, heads, length, dim, kv_heads, page, kernel, kernel2, length > 1)
    batch = round(32 ** rng.random())
    most = min(65536, (LIMIT >> (1 if dtype == "fp32" else 0)) // (2 * token * batch))
    # long rows of wide kernels are what the plain form's windows take memory for
    most = max(32, min(most, (1 << 31) // (batch * heads * kernel[0] * kernel[1] * (kernel2[0] if op == "mta" else 1) * 4)))
    length = round(16 * (most / 16) ** rng.random())
    return _case(None, op, dtype, batch, heads, length, dim, kv_heads, page, kernel, kernel2, rng.random() < 0.7)


def _lengths(case):
    """Tokens of each sequence (append: new tokens), spread over the upper part of the range: part of the case, not of the inputs."""
    n, b = case["length"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    r = random.Random("%d %d %d %d" % (n, b, case["heads"], case["dim"]))
    return [n] + [r.randint(max(1, n // 4), n) for _ in range(b - 1)]


def _rows(case):
    """Queries that one new token looks at: its own and those that the convs reach back to."""
    return case["cq"] + (case["cq2"] if case["op"] != "conv" else 1) - 1


def _earlier(case):
    """append: tokens that each sequence has already, so that the new ones begin inside a page."""
    return 37 if case["length"] > 1 else 1000


def _conv_kernel(g, heads, rows, cols):
    w = torch.randn(heads, rows, cols, device="cuda", generator=g) * (rows * cols) ** -0.5
    w[:, rows - 1, cols // 2] += 1.0
    return w


def _mix(g, heads):
    return torch.eye(heads, device="cuda") + 0.02 ** 0.5 * torch.randn(heads, heads, device="cuda", generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = DTYPES[case["dtype"]], case["op"]
    h, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)

    rows = _rows(case)
    if op == "copy":
        # the pages in use lie anywhere in the pool: a permutation gives sources and destinations that never meet
        n = case["length"]
        pool = 2 * n + n // 8
        perm = torch.randperm(pool, device="cuda", generator=g)
        return {"op": op, "k_pages": normal(pool, hk, page, d), "v_pages": normal(pool, hk, page, d),
                "src": perm[:n].int().contiguous(), "dst": perm[n:2 * n].int().contiguous()}
    lens = _lengths(case)
    before = _earlier(case) if op == "append" else 0
    total = [n + before for n in lens]
    pages = [-(-n // page) for n in total]
    pool = sum(pages) + 8
    perm = torch.randperm(pool, device="cuda", generator=g).int()
    table = torch.zeros(len(lens), max(pages), device="cuda", dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    state = {"op": op, "k_pages": normal(pool, hk, page, d), "v_pages": normal(pool, hk, page, d),
             "q_hist": normal(len(lens), rows, h, d), "table": table, "lengths": torch.tensor(total, device="cuda", dtype=torch.int32)}
    if op == "append":
        t = case["length"]
        state |= {"k": normal(len(lens), hk, t, d), "v": normal(len(lens), hk, t, d), "q": normal(len(lens), h, t, d),
                  "counts": torch.tensor(lens, device="cuda", dtype=torch.int32)}
        return state
    state |= {"max_length": max(total), "w1": _conv_kernel(g, h, case["cq"], case["ck"]).to(dtype), "scale": d ** -0.5}
    if op == "mta":
        state |= {"W1": _mix(g, h).to(dtype), "w2": _conv_kernel(g, h, case["cq2"], case["ck2"]).to(dtype), "W2": _mix(g, h).to(dtype)}
    return state


def _dense(pages, table, lengths, heads):
    """(batch, heads, keys, dim) in float32, zeros behind each sequence's end."""
    b, n = table.shape
    _, hk, page, d = pages.shape
    x = pages[table.long()].permute(0, 2, 1, 3, 4).reshape(b, hk, n * page, d).float()
    live = torch.arange(n * page, device=x.device)[None, :] < lengths[:, None]
    x = torch.where(live[:, None, :, None], x, torch.zeros((), device=x.device))
    return x if hk == heads else x[:, torch.arange(heads, device=x.device) // (heads // hk)]


def _conv(x, w):
    """Depthwise conv over (batch, heads, rows, keys): the taps' last row on the row itself, the keys centred; rows that have all their taps."""
    cq, ck = w.shape[1:]
    left = (ck - 1) // 2
    z = torch.zeros(*x.shape[:3], ck - 1, device=x.device)
    x = torch.cat([z[..., :left], x, z[..., left:]], dim=3)
    windows = x.unfold(2, cq, 1).unfold(3, ck, 1)
    return torch.einsum("bhrsij,hij->bhrs", windows, w.float())


def _plain_attention(state):
    q_hist, table, lengths = state["q_hist"], state["table"], state["lengths"].long()
    b, ring, heads, d = q_hist.shape
    w1 = state["w1"]
    mta = state["op"] == "mta"
    cq2 = state["w2"].shape[1] if mta else 1
    rows = w1.shape[1] + cq2 - 1
    dev = q_hist.device
    pos = lengths[:, None] - rows + torch.arange(rows, device=dev)                  # (batch, rows)
    q = q_hist[torch.arange(b, device=dev)[:, None], pos % ring].permute(0, 2, 1, 3).float()
    k = _dense(state["k_pages"], table, lengths, heads)
    v = _dense(state["v_pages"], table, lengths, heads)
    key = torch.arange(k.shape[2], device=dev)
    seen = (key <= pos[:, :, None])[:, None]                                        # rows before the first token see no key
    zero, low = torch.zeros((), device=dev), torch.full((), -math.inf, device=dev)
    s = torch.where(seen, torch.matmul(q, k.transpose(2, 3)) * state["scale"], zero)
    c = _conv(s, w1)
    seen = seen[:, :, rows - cq2:]
    if mta:
        c = torch.einsum("oh,bhrs->bors", state["W1"].float(), c)
    c = torch.where(seen, c, low)
    e = torch.where(seen, torch.exp(c - c.amax(dim=3, keepdim=True)), zero)
    p = e / e.sum(dim=3, keepdim=True)
    if mta:
        p = torch.where(seen, p, zero)
        p = torch.where(seen[:, :, cq2 - 1:], _conv(p, state["w2"]), zero)
        p = torch.einsum("oh,bhrs->bors", state["W2"].float(), p)
    return torch.matmul(p, v).to(q_hist.dtype)


def _plain_append(state):
    k, table, lengths, counts = state["k"], state["table"].long(), state["lengths"].long(), state["counts"].long()
    b, _, t, _ = k.shape
    dev = k.device
    page, ring = state["k_pages"].shape[2], state["q_hist"].shape[1]
    row = torch.arange(b, device=dev)[:, None]
    # tokens behind a sequence's last are its last again: the same value to the same place
    token = torch.minimum(torch.arange(t, device=dev)[None, :], counts[:, None] - 1)
    pos = lengths[:, None] - counts[:, None] + token
    at, slot = table[row, pos // page], pos % page
    state["k_pages"][at, :, slot] = k[row, :, token]
    state["v_pages"][at, :, slot] = state["v"][row, :, token]
    token = torch.clamp(counts[:, None] - ring + torch.arange(ring, device=dev), min=0)
    pos = lengths[:, None] - counts[:, None] + token
    state["q_hist"][row, pos % ring] = state["q"][row, :, token]


def run(state):
    op = state["op"]
    if own:
        from multitokenatention_triton_b200 import ops
    if op == "copy":
        if own:
            ops.cache_copy(state["k_pages"], state["v_pages"], state["src"], state["dst"])
        else:
            src, dst = state["src"].long(), state["dst"].long()
            state["k_pages"][dst] = state["k_pages"][src]
            state["v_pages"][dst] = state["v_pages"][src]
        return [state["k_pages"], state["v_pages"]]
    if op == "append":
        if own:
            ops.cache_append(state["k"], state["v"], state["q"], state["k_pages"], state["v_pages"], state["q_hist"], state["table"],
                             state["lengths"], counts=state["counts"])
        else:
            _plain_append(state)
        return [state["k_pages"], state["v_pages"], state["q_hist"]]
    if not own:
        return _plain_attention(state)
    cache = (state["q_hist"], state["k_pages"], state["v_pages"], state["table"], state["lengths"])
    if op == "mta":
        return ops.mta_decode_fwd(*cache, state["w1"], state["W1"], state["w2"], state["W2"], state["max_length"])
    return ops.conv_attn_decode_fwd(*cache, state["w1"], state["scale"], state["max_length"])


def work(case):
    h, hk, d, e = case["heads"], case["kv_heads"], case["dim"], SIZE[case["dtype"]]
    op, rows = case["op"], _rows(case)
    if op == "copy":
        return {"bytes": case["length"] * (4 * hk * case["page"] * d * e + 8), "flops": 0}
    lens = _lengths(case)
    if op == "append":
        return {"bytes": sum(2 * e * d * (2 * hk * n + h * min(n, rows)) for n in lens) + 12 * len(lens), "flops": 0}
    taps, taps2 = case["cq"] * case["ck"], case["cq2"] * case["ck2"]
    if op == "mta":
        per = 2 * d * rows + 2 * taps * case["cq2"] + 2 * h * case["cq2"] + 2 * taps2 + 2 * h + 2 * d
        weights = h * (taps + taps2 + 2 * h)
    else:
        per, weights = 2 * d * rows + 2 * taps + 2 * d, h * taps
    return {"bytes": sum(2 * hk * n * d * e + (rows + 1) * h * d * e + 4 * -(-n // case["page"]) for n in lens) + weights * e,
            "flops": per * h * sum(lens)}


def _conv64(x, w):
    """The conv of one sequence's rows (heads, rows, keys) in float64, tap by tap."""
    heads, cq, ck = w.shape
    n, keys, left = x.shape[1] - cq + 1, x.shape[2], (ck - 1) // 2
    y = torch.zeros(heads, n, keys, device=x.device, dtype=torch.float64)
    for j in range(ck):
        a, z = max(0, left - j), min(keys, keys + left - j)      # keys whose neighbour at this tap lies inside the plane
        if a < z:
            for i in range(cq):
                y[:, :, a:z] += w[:, i, j, None, None] * x[:, i:i + n, a + j - left:z + j - left]
    return y


def exact(case, seed):
    if case["op"] in ("append", "copy"):
        return None                                              # values are moved, none is computed
    state = prepare(case, seed)
    out = []
    page, group = case["page"], case["heads"] // case["kv_heads"]
    w1 = state["w1"].double()
    for b, n in enumerate(_lengths(case)):
        at = state["table"][b, :-(-n // page)].long()
        k, v = (torch.cat([state[name][at, i].reshape(1, -1, case["dim"])[:, :n].double() for i in range(case["kv_heads"])])
                for name in ("k_pages", "v_pages"))
        rows = _rows(case)
        score = torch.zeros(case["heads"], rows, n, device="cuda", dtype=torch.float64)
        for r in range(rows):
            p = n - rows + r
            if p >= 0:
                q = state["q_hist"][b, p % state["q_hist"].shape[1]].double()
                for h in range(case["heads"]):
                    score[h, r, :p + 1] = k[h // group, :p + 1] @ q[h] / math.sqrt(case["dim"])
        x = _conv64(score, w1)
        if case["op"] == "mta":
            x = torch.tensordot(state["W1"].double(), x, dims=1)
        prob = torch.zeros_like(x)
        for r in range(x.shape[1]):
            p = n - x.shape[1] + r
            if p >= 0:
                prob[:, r, :p + 1] = torch.softmax(x[:, r, :p + 1], dim=1)
        if case["op"] == "mta":
            prob = torch.tensordot(state["W2"].double(), _conv64(prob, state["w2"].double()), dims=1)
        out.append(torch.stack([prob[h] @ v[h // group] for h in range(case["heads"])]))
    return torch.stack(out)
