"""Cases of the full-rank paged cache's operators: what writes it, what reads it, and
what reads only the pages that matter.

    decode   one new token per sequence over a paged K/V cache
    write    per-head norms of queries and keys, the rotation, and the write into the cache
    bounds   per-page lower / upper bounds of the keys
    sparse   the pages that the bounds select for each query, and the attention over them

``own = False`` computes them with elementary torch operations, ``own = True`` through
``starkv_b200.kernels``. The geometry is this repository's (32 heads of 128, 4096 hidden,
pages of 16, contexts of 8192 to 32768, batches of 24 and 64) and grouped variants of it.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def kernels():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "star-kv-serve_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from starkv_b200.kernels import paged_attention, qk_norm_rope
    return paged_attention, qk_norm_rope


# ----------------------------------------------------------------------------- cases

def listed():
    return [
        # one chat turn at a short context: a call of a few microseconds, where latency counts
        {"name": "decode_one_short", "op": "decode", "n": 1, "lo": 201, "hi": 201, "heads": 32, "kv": 8, "dim": 128,
         "block": 16, "dtype": "bf16", "order": "head", "partial": False},
        # a serving batch of ragged sequences (one of them empty: a padded row of a captured step), grouped heads
        {"name": "decode_ragged_grouped", "op": "decode", "n": 33, "lo": 0, "hi": 8191, "heads": 32, "kv": 8,
         "dim": 128, "block": 16, "dtype": "f16", "order": "token", "partial": False},
        # the model's full-rank layers: 24 sessions, 32 query and 32 key heads
        {"name": "decode_mha_24x8192", "op": "decode", "n": 24, "lo": 8192, "hi": 8192, "heads": 32, "kv": 32,
         "dim": 128, "block": 16, "dtype": "bf16", "order": "head", "partial": False},
        # one long document, few rows: the length has to be split over the whole GPU; one rank's share of a
        # page split, which returns what the ranks' combine takes
        {"name": "decode_one_long_partial", "op": "decode", "n": 1, "lo": 131071, "hi": 131071, "heads": 32, "kv": 8,
         "dim": 128, "block": 64, "dtype": "bf16", "order": "head", "partial": True},
        # one new token: the smallest write
        {"name": "write_one", "op": "write", "n": 1, "heads": 32, "kv": 8, "dim": 128, "block": 16, "dtype": "bf16",
         "norm": True, "order": "head", "table": "bf16", "pad": 0},
        # a decode step of 64 sequences without norms (the model's own rotary), some rows padding
        {"name": "write_step_64", "op": "write", "n": 64, "heads": 32, "kv": 32, "dim": 128, "block": 16,
         "dtype": "bf16", "norm": False, "order": "head", "table": "bf16", "pad": 3},
        # prompts of a prefill with norms, an odd number of tokens
        {"name": "write_prefill_8191", "op": "write", "n": 8191, "heads": 32, "kv": 8, "dim": 128, "block": 16,
         "dtype": "f16", "norm": True, "order": "token", "table": "f32", "pad": 0},
        # after a decode step: the page of each sequence's new token
        {"name": "bounds_step_64", "op": "bounds", "n": 64, "lo": 1024, "hi": 8191, "kv": 8, "dim": 128, "block": 16,
         "dtype": "bf16", "order": "head", "new": 1},
        # after a prefill: every page of the prompts
        {"name": "bounds_prefill_8x8190", "op": "bounds", "n": 8, "lo": 4097, "hi": 8190, "kv": 8, "dim": 128,
         "block": 16, "dtype": "bf16", "order": "token", "new": 8190},
        # one long document, 64 of its 8192 pages
        {"name": "sparse_one_131071", "op": "sparse", "n": 1, "lo": 131071, "hi": 131071, "heads": 32, "kv": 8,
         "dim": 128, "block": 16, "dtype": "bf16", "order": "head", "top": 64},
        # a batch of long sessions, 64 pages each
        {"name": "sparse_64_to_32768", "op": "sparse", "n": 64, "lo": 1024, "hi": 32768, "heads": 32, "kv": 8,
         "dim": 128, "block": 16, "dtype": "bf16", "order": "head", "top": 64},
        # shorter sequences, some with fewer pages than are asked for; larger pages, small heads
        {"name": "sparse_16_small_heads", "op": "sparse", "n": 16, "lo": 300, "hi": 9000, "heads": 8, "kv": 2,
         "dim": 64, "block": 32, "dtype": "f16", "order": "token", "top": 33},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "write", "bounds", "sparse"])
    kv = rng.choice([1, 2, 4, 8, 32])
    heads = kv * rng.choice([1] if kv == 32 else [1, 2, 4, 5, 8])
    c = {"op": op, "kv": kv, "dim": rng.choice([64, 128, 128]), "block": rng.choice([16, 16, 32, 64]),
         "dtype": rng.choice(["bf16", "f16"]), "order": rng.choice(["head", "token"])}
    if op == "write":
        c |= {"n": _log(rng, 1, 8191), "heads": heads, "norm": rng.random() < 0.6, "table": rng.choice(["bf16", "f32"]),
              "pad": 0}
        c["pad"] = rng.randrange(0, 1 + c["n"] // 8)
        return c
    n = _log(rng, 1, 64)
    # at most the tokens x heads of the largest listed case of the kind
    most = {"decode": 24 * 8192 * 32, "bounds": 8 * 8190 * 8, "sparse": 64 * 16896 * 8}[op] // (n * kv)
    hi = _log(rng, 2, max(2, min(131071, most)))
    lo = rng.choice([hi, hi // 2, min(hi, 1)])
    c |= {"n": n, "lo": lo, "hi": hi}
    if op == "bounds":
        return c | {"new": rng.choice([1, 1, hi])}
    c["heads"] = heads
    return c | ({"partial": rng.random() < 0.25} if op == "decode" else {"top": _log(rng, 3, 128)})


# ----------------------------------------------------------------------------- inputs

def _lens(case, gen):
    n, lo, hi = case["n"], case["lo"], case["hi"]
    v = torch.randint(lo, hi + 1, (n,), generator=gen, device="cuda")
    v[0] = hi
    if lo == 0 and n > 1:
        v[n // 2] = 0
    return v.int()


def _cache(case, blocks, gen, spread=True):
    """[blocks, block, kv, dim] in the asked order of heads and tokens; channels of a key head differ in size and
    mean, as rotated keys' do, so that some pages score above others."""
    kv, D, bs, dt = case["kv"], case["dim"], case["block"], DTYPES[case["dtype"]]
    if case["order"] == "head":
        t = torch.empty(blocks, kv, bs, D, dtype=dt, device="cuda").transpose(1, 2)
    else:
        t = torch.empty(blocks, bs, kv, D, dtype=dt, device="cuda")
    t.normal_(generator=gen)
    if spread:
        t.mul_((0.5 + torch.rand(kv, D, generator=gen, device="cuda")).to(dt))
        t.add_(torch.randn(blocks, 1, kv, 1, generator=gen, device="cuda").to(dt) * 0.25)
    return t


def _tables(case, lens, gen):
    bs = case["block"]
    per = max(1, -(-case["hi"] // bs))
    blocks = case["n"] * per + 1     # block 0 is the null block
    bt = (torch.randperm(blocks - 1, generator=gen, device="cuda")[:case["n"] * per] + 1).view(case["n"], per).int()
    return bt, blocks


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    dt, D, kv, bs, n = DTYPES[case["dtype"]], case["dim"], case["kv"], case["block"], case["n"]
    s = dict(case)
    if case["op"] == "write":
        H = case["heads"]
        qkv = torch.randn(n, H + 2 * kv, D, generator=gen, device="cuda").mul_(1.5).to(dt)
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + kv], qkv[:, H + kv:]
        blocks = -(-n // bs) + 2
        slots = torch.randperm((blocks - 1) * bs, generator=gen, device="cuda")[:n] + bs
        if case["pad"]:
            slots[n - case["pad"]:] = -1
        s["slots"] = slots
        s["k_cache"], s["v_cache"] = _cache(case, blocks, gen, False), _cache(case, blocks, gen, False)
        rows = 32768
        s["positions"] = torch.randint(0, rows, (n,), generator=gen, device="cuda")
        inv = 1.0 / (10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D))
        ang = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
        table = torch.cat([ang.cos(), ang.sin()], 1)
        s["cos_sin"] = table.to(torch.float32 if case["table"] == "f32" else torch.bfloat16)
        s["q_weight"] = s["k_weight"] = None
        if case["norm"]:
            s["q_weight"] = (1 + 0.1 * torch.randn(D, generator=gen, device="cuda")).to(dt)
            s["k_weight"] = (1 + 0.1 * torch.randn(D, generator=gen, device="cuda")).to(dt)
        return s
    s["lens"] = _lens(case, gen)
    s["bt"], blocks = _tables(case, s["lens"], gen)
    s["k_cache"] = _cache(case, blocks, gen)
    if case["op"] == "bounds":
        s["bounds"] = torch.zeros(blocks, kv, 2, D, dtype=dt, device="cuda")
        return s
    s["v_cache"] = _cache(case, blocks, gen, False)
    s["q"] = torch.randn(n, case["heads"], D, generator=gen, device="cuda").mul_(1.7).to(dt)
    s["scale"] = D ** -0.5
    if case["op"] == "sparse":   # kept up to date page by page as the cache is written
        s["bounds"] = torch.stack([s["k_cache"].amin(1), s["k_cache"].amax(1)], 2)
    return s


# ----------------------------------------------------------------------------- one pass

def run(s):
    return {"decode": _decode, "write": _write, "bounds": _bounds, "sparse": _sparse}[s["op"]](s)


def _attend(q, K, V, valid, scale):
    """q [n, H, D], K and V [n, kv, T, D], valid [n, kv or 1, T] -> (out, max, denominator) in f32, out not divided."""
    n, H, D = q.shape
    kv = K.shape[1]
    qf = q.float().view(n, kv, H // kv, D)
    logit = torch.matmul(qf, K.float().transpose(2, 3)) * scale
    logit = logit.masked_fill(~valid[:, :, None, :], float("-inf"))
    m = logit.amax(-1, keepdim=True)
    p = torch.exp(logit - torch.where(m.isinf(), torch.zeros_like(m), m))
    return torch.matmul(p, V.float()).view(n, H, D), m.view(n, H), p.sum(-1).view(n, H)


def _divided(out, l, dtype):
    return torch.where(l[..., None] > 0, out / l[..., None], torch.zeros_like(out)).to(dtype)


def _decode(s):
    if own:
        pa, _ = kernels()
        return pa.paged_attention_decode(s["q"], s["k_cache"], s["v_cache"], s["bt"], s["lens"], s["hi"], s["scale"],
                                         return_partial=s["partial"])
    n, D, kv = s["n"], s["dim"], s["kv"]
    at = s["bt"].long()
    K = s["k_cache"][at].reshape(n, -1, kv, D).transpose(1, 2)
    V = s["v_cache"][at].reshape(n, -1, kv, D).transpose(1, 2)
    valid = torch.arange(K.shape[2], device=K.device) < s["lens"][:, None]
    V = V.masked_fill(~valid[:, None, :, None], 0)
    out, m, l = _attend(s["q"], K, V, valid[:, None], s["scale"])
    return (out, m, l) if s["partial"] else _divided(out, l, s["q"].dtype)


def _rotated(x, weight, cos, sin):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _write(s):
    if own:
        _, nr = kernels()
        q = nr.qk_norm_rope_write(s["q"], s["k"], s["v"], s["positions"], s["cos_sin"], s["k_cache"], s["v_cache"],
                                  s["slots"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
        return q, s["k_cache"], s["v_cache"]
    cos, sin = s["cos_sin"][s["positions"]].float()[:, None].chunk(2, -1)
    q = _rotated(s["q"], s["q_weight"], cos, sin).to(s["q"].dtype)
    k = _rotated(s["k"], s["k_weight"], cos, sin).to(s["k"].dtype)
    real = s["n"] - s["pad"]
    at = s["slots"][:real]
    s["k_cache"][at // s["block"], at % s["block"]] = k[:real]
    s["v_cache"][at // s["block"], at % s["block"]] = s["v"][:real]
    return q, s["k_cache"], s["v_cache"]


def _bounds(s):
    if own:
        pa, _ = kernels()
        pa.update_page_bounds(s["k_cache"], s["bounds"], s["bt"], s["lens"], s["hi"], max_new=s["new"])
        return s["bounds"]
    bs, lens = s["block"], s["lens"].long()[:, None]
    page = torch.arange(s["bt"].shape[1], device=lens.device)
    first = (lens - s["new"]).clamp(min=0) // bs
    row, col = torch.nonzero((page >= first) & (page * bs < lens), as_tuple=True)
    at = s["bt"].long()[row, col]
    K = s["k_cache"][at]
    inside = (col[:, None] * bs + torch.arange(bs, device=lens.device) < lens[row])[:, :, None, None]
    s["bounds"][at, :, 0] = K.masked_fill(~inside, float("inf")).amin(1)
    s["bounds"][at, :, 1] = K.masked_fill(~inside, float("-inf")).amax(1)
    return s["bounds"]


def _sparse(s):
    if own:
        pa, _ = kernels()
        return pa.sparse_paged_decode(s["q"], s["k_cache"], s["v_cache"], s["bounds"], s["bt"], s["lens"], s["hi"],
                                      s["scale"], s["top"])
    n, H, D, kv, bs, top = s["n"], s["heads"], s["dim"], s["kv"], s["block"], s["top"]
    lens = s["lens"].long()
    at = s["bt"].long()
    P = at.shape[1]
    pages = (lens + bs - 1) // bs
    # scores in 64 bits: the order of two pages next to the border has to come out the same
    qd = s["q"].double().view(n, kv, H // kv, D)
    up, down = qd.clamp(min=0).sum(2)[..., None], qd.clamp(max=0).sum(2)[..., None]
    B = s["bounds"][at].transpose(1, 2).double()
    score = (torch.matmul(B[:, :, :, 1], up) + torch.matmul(B[:, :, :, 0], down))[..., 0]
    col = torch.arange(P, device=at.device)
    real = (col < pages[:, None])[:, None].expand(n, kv, P)
    kept = ((col < 1) | (col >= pages[:, None] - 1))[:, None]
    score = score.masked_fill(kept, float("inf")).masked_fill(~real, float("-inf"))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    order = torch.where(order < pages[:, None, None], order, P).sort(-1).values
    picked = torch.full((n, kv, top), -1, dtype=torch.int32, device=at.device)
    picked[..., :order.shape[-1]] = torch.where(order < P, order, -1)
    page = picked.long().clamp(min=0)
    block = torch.gather(at[:, None].expand(n, kv, P), 2, page)
    head = torch.arange(kv, device=at.device)[None, :, None]
    K = s["k_cache"].transpose(1, 2)[block, head].reshape(n, kv, top * bs, D)
    V = s["v_cache"].transpose(1, 2)[block, head].reshape(n, kv, top * bs, D)
    pos = page[..., None] * bs + torch.arange(bs, device=at.device)
    valid = ((pos < lens[:, None, None, None]) & (picked >= 0)[..., None]).view(n, kv, top * bs)
    V = V.masked_fill(~valid[..., None], 0)
    out, _, l = _attend(s["q"], K, V, valid, s["scale"])
    return _divided(out, l, s["q"].dtype), picked


# ----------------------------------------------------------------------------- cost

def _tokens(case):
    """Expected tokens of the batch (the lengths are uniform over lo .. hi, the first is hi)."""
    return case["hi"] + (case["n"] - 1) * (case["lo"] + case["hi"]) / 2


def work(case):
    n, kv, D, e = case["n"], case["kv"], case["dim"], 2
    if case["op"] == "write":
        H = case["heads"]
        table = n * D * (4 if case["table"] == "f32" else 2)
        return {"bytes": 2 * n * (H + 2 * kv) * D * e + table + 16 * n, "flops": 8 * n * (H + kv) * D}
    T, bs = _tokens(case), case["block"]
    if case["op"] == "bounds":
        tokens = min(T, n * min(case["new"], case["hi"]) + n * (bs - 1) / 2)
        return {"bytes": tokens * kv * D * e + (tokens / bs + n / 2) * kv * 2 * D * e, "flops": 2 * tokens * kv * D}
    H = case["heads"]
    io = n * H * D * (e + (4 if case.get("partial") else e)) + (8 * n * H if case.get("partial") else 0)
    if case["op"] == "decode":
        return {"bytes": 2 * T * kv * D * e + io + 4 * T / bs, "flops": 4 * T * H * D}
    pages = T / bs + n / 2
    read = min(T, n * case["top"] * bs)
    return {"bytes": pages * kv * 2 * D * e + 2 * read * kv * D * e + io + 4 * pages + 4 * n * kv * case["top"],
            "flops": 4 * pages * kv * D + 4 * read * H * D}


# ----------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    f = {"decode": _exact_decode, "write": _exact_write, "bounds": _exact_bounds, "sparse": _exact_sparse}
    return f[case["op"]](s)


def _softmax64(q, K, V, scale):
    """q [H, D], K and V [T, kv, D] in 64 bits, T >= 1."""
    g = q.shape[0] // K.shape[1]
    K, V = K.repeat_interleave(g, 1), V.repeat_interleave(g, 1)
    x = scale * (K * q).sum(-1)
    m = x.max(0).values
    w = torch.exp(x - m)
    return (w[..., None] * V).sum(0), m, w.sum(0)


def _exact_decode(s):
    out = torch.zeros(s["n"], s["heads"], s["dim"], dtype=torch.float64, device="cuda")
    m = torch.full(out.shape[:2], float("-inf"), dtype=torch.float64, device="cuda")
    l = torch.zeros_like(m)
    for b, L in enumerate(s["lens"].tolist()):
        if not L:
            continue
        ids = s["bt"][b, :-(-L // s["block"])].long()
        for h in range(s["kv"]):   # a KV head at a time bounds the memory
            g = s["heads"] // s["kv"]
            K = s["k_cache"][ids, :, h:h + 1].reshape(-1, 1, s["dim"])[:L].double()
            V = s["v_cache"][ids, :, h:h + 1].reshape(-1, 1, s["dim"])[:L].double()
            r = slice(h * g, (h + 1) * g)
            out[b, r], m[b, r], l[b, r] = _softmax64(s["q"][b, r].double(), K, V, s["scale"])
    if s["partial"]:
        return out, m, l
    return out / torch.where(l > 0, l, torch.ones_like(l))[..., None]


def _exact_write(s):
    tab = s["cos_sin"][s["positions"]].double()
    half = s["dim"] // 2
    z = torch.complex(tab[:, :half], tab[:, half:])[:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / s["dim"] + EPS) * w.double()
        y = torch.complex(x[..., :half], x[..., half:]) * z
        return torch.cat([y.real, y.imag], -1)

    K, V = s["k_cache"].double(), s["v_cache"].double()
    k = turned(s["k"], s["k_weight"])
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    K[at // s["block"], at % s["block"]] = k[keep]
    V[at // s["block"], at % s["block"]] = s["v"][keep].double()
    return turned(s["q"], s["q_weight"]), K, V


def _exact_bounds(s):
    out = s["bounds"].double()
    bs = s["block"]
    for b, L in enumerate(s["lens"].tolist()):
        for p in range(max(0, L - s["new"]) // bs, -(-L // bs)):
            blk = int(s["bt"][b, p])
            rows = s["k_cache"][blk, :min(bs, L - p * bs)].double()
            out[blk, :, 0], out[blk, :, 1] = rows.min(0).values, rows.max(0).values
    return out


def _exact_sparse(s):
    n, H, D, kv, bs, top = s["n"], s["heads"], s["dim"], s["kv"], s["block"], s["top"]
    out = torch.zeros(n, H, D, dtype=torch.float64, device="cuda")
    picked = torch.full((n, kv, top), -1, dtype=torch.int32, device="cuda")
    g = H // kv
    for b, L in enumerate(s["lens"].tolist()):
        P = -(-L // bs)
        if not P:
            continue
        ids = s["bt"][b, :P].long()
        B = s["bounds"][ids].double()
        for h in range(kv):
            q = s["q"][b, h * g:(h + 1) * g].double()
            x = torch.maximum(q[:, None] * B[None, :, h, 0], q[:, None] * B[None, :, h, 1]).sum((0, 2))
            x[0] = x[P - 1] = float("inf")
            best = torch.argsort(x, descending=True, stable=True)[:top].sort().values
            picked[b, h, :best.numel()] = best
            K = s["k_cache"][ids[best], :, h:h + 1].double()
            V = s["v_cache"][ids[best], :, h:h + 1].double()
            inside = (best[:, None] * bs + torch.arange(bs, device="cuda")) < L
            o, _, l = _softmax64(q, K[inside], V[inside], s["scale"])
            out[b, h * g:(h + 1) * g] = o / l[..., None]
    return out, picked
