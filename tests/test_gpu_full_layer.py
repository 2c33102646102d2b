"""GPU checks of the full-rank layer (starkv_b200.full_layer) and of the model that uses it:
the cache's operators run together - norm + rotary + write, page bounds, selection, decode,
prefill - against a dense float32 recomputation of the layer on the same weights, and the
page split against the whole layer.

Tolerances: a layer's output is compared in norm. The projections round q, k, v, the
attention and the output to bf16 (2^-8 relative at most each, about 2^-9.8 on average);
five such steps in a row stay under 5 2^-8 = 2e-2 of the norm.
"""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

HID, D = 512, 128


def cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda", 0)


def weights(H, Hkv, seed=0, norm=True):
    dev = cuda()
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g, device=dev) * s[-1] ** -0.5).to(torch.bfloat16)  # noqa: E731
    w = [r(H * D, HID), r(Hkv * D, HID), r(Hkv * D, HID), r(HID, H * D)]
    qn, kn = ((1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16) for _ in range(2))
    from starkv_b200.workload import rope_cos_sin
    return w, (dict(q_norm=qn, k_norm=kn) if norm else {}), rope_cos_sin(4096, dev)


def dense(w, norms, cs, hidden, eps=1e-6):
    """float32 layer on one whole sequence hidden [T, HID] -> [T, HID], causal."""
    T = hidden.shape[0]
    wq, wk, wv, wo = (t.float() for t in w)
    q, k, v = (F.linear(hidden.float(), t).view(T, -1, D) for t in (wq, wk, wv))
    if norms:
        n = lambda x, g: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * g.float()  # noqa: E731
        q, k = n(q, norms["q_norm"]), n(k, norms["k_norm"])
    c, s = cs[:T].float()[:, None].chunk(2, -1)
    turn = lambda x: torch.cat([x[..., :64] * c - x[..., 64:] * s, x[..., 64:] * c + x[..., :64] * s], -1)  # noqa: E731
    G = q.shape[1] // k.shape[1]
    q, k, v = turn(q), turn(k).repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    a = torch.einsum("thd,shd->hts", q, k) * D ** -0.5
    a = a.masked_fill(~torch.ones(T, T, dtype=torch.bool, device=a.device).tril(), float("-inf")).softmax(-1)
    return F.linear(torch.einsum("hts,shd->thd", a, v).reshape(T, -1), wo)


def rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


@pytest.mark.parametrize("H,Hkv,norm", [(4, 4, False), (8, 2, True)])
@pytest.mark.parametrize("top", [None, 64])
def test_prefill_then_decode_matches_the_dense_layer(H, Hkv, norm, top):
    """Prompts of several lengths, then steps that cross a page border, one row of padding."""
    from starkv_b200.full_layer import FullAttentionLayer
    w, norms, cs = weights(H, Hkv, seed=H, norm=norm)
    dev = cs.device
    layer = FullAttentionLayer(*w, cs, top_pages=top, **norms)
    lens, steps, per = [30, 1, 127], 5, 9
    bt = (torch.randperm(4 * per, device=dev).view(4, per) + 1).int()
    cache = layer.allocate_cache(4 * per + 1)
    for c in cache:
        c.fill_(float("nan"))                              # nothing unwritten may show
    g = torch.Generator(device=dev).manual_seed(3)
    seqs = [torch.randn(L + steps, HID, generator=g, device=dev).to(torch.bfloat16) for L in lens]
    want = [dense(w, norms, cs, s) for s in seqs]
    slot = lambda b, t: bt[b, t // 16].long() * 16 + t % 16  # noqa: E731
    pos = torch.cat([torch.arange(L, device=dev) for L in lens])
    slots = torch.cat([slot(b, torch.arange(L, device=dev)) for b, L in enumerate(lens)])
    out = layer.prefill(torch.cat([s[:L] for s, L in zip(seqs, lens)]), pos, lens, cache, slots, block_table=bt[:3])
    assert rel(out, torch.cat([x[:L] for x, L in zip(want, lens)])) < 2e-2
    for i in range(steps):
        hidden = torch.stack([s[L + i] for s, L in zip(seqs, lens)] + [torch.ones_like(seqs[0][0])])
        p = torch.tensor([L + i for L in lens] + [0], device=dev)
        sl = torch.tensor([L + i + 1 for L in lens] + [0], dtype=torch.int32, device=dev)
        sm = torch.stack([slot(b, torch.tensor(L + i, device=dev)) for b, L in enumerate(lens)]
                         + [torch.tensor(-1, device=dev)])
        out = layer.forward(hidden, p, cache, bt, sl, per * 16, sm)
        assert rel(out[:3], torch.stack([x[L + i] for x, L in zip(want, lens)])) < 2e-2
        assert (out[3] == 0).all()


def test_selected_pages_are_what_the_operators_give():
    """With fewer pages than the sequence has: the layer is its operators called one by one."""
    from starkv_b200.full_layer import FullAttentionLayer
    from starkv_b200.kernels import paged_attention as pa
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope
    w, norms, cs = weights(8, 2, seed=1)
    dev = cs.device
    layer = FullAttentionLayer(*w, cs, top_pages=6, **norms)
    T, per = 700, 44
    bt = (torch.randperm(per, device=dev)[None] + 1).int()
    cache = layer.allocate_cache(per + 1)
    hidden = torch.randn(T + 1, HID, device=dev).to(torch.bfloat16)
    t = torch.arange(T + 1, device=dev)
    slots = bt[0, t // 16].long() * 16 + t % 16
    layer.prefill(hidden[:T], t[:T], [T], cache, slots[:T], block_table=bt)
    sl = torch.tensor([T + 1], dtype=torch.int32, device=dev)
    out = layer.forward(hidden[T:], t[T:], cache, bt, sl, 704, slots[T:])
    q = F.linear(hidden[T:], layer.wqkv).view(1, 12, D)[:, :8]
    q, _ = qk_norm_rope(q, None, t[T:], cs, q_weight=norms["q_norm"])
    rows = cache[0][bt[0].long()].reshape(-1, 2, D)[:T + 1]
    pad = F.pad(rows, (0, 0, 0, 0, 0, 704 - T - 1), value=float("nan")).view(44, 16, 2, D)
    lo = torch.nan_to_num(pad, nan=float("inf")).amin(1)
    assert torch.equal(cache[2][bt[0].long(), :, 0], lo)
    attn, pages = pa.sparse_paged_decode(q, *cache, bt, sl, 704, D ** -0.5, 6)
    assert torch.equal(out, F.linear(attn.view(1, -1), layer.wo))
    assert pages.shape == (1, 2, 6) and (pages[..., 0] == 0).all() and (pages[..., -1] == 43).all()


def test_head_shards_sum_to_the_whole_layer():
    from starkv_b200.full_layer import FullAttentionLayer
    w, norms, cs = weights(8, 4, seed=2)
    dev = cs.device
    bt = torch.arange(1, 9, device=dev, dtype=torch.int32).view(2, 4)
    outs = []
    for world in (1, 2, 4):
        total = 0
        for r in range(world):
            layer = FullAttentionLayer(*w, cs, rank=r, world=world, **norms)
            cache = layer.allocate_cache(9)
            g = torch.Generator(device=dev).manual_seed(7)
            for t in range(20):
                hidden = torch.randn(2, HID, generator=g, device=dev).to(torch.bfloat16)
                slots = bt[:, t // 16].long() * 16 + t % 16
                out = layer.forward(hidden, torch.full((2,), t, device=dev), cache, bt,
                                    torch.full((2,), t + 1, dtype=torch.int32, device=dev), 64, slots, reduce=False)
            total = total + out.float()
        outs.append(total)
    assert rel(outs[1], outs[0]) < 1e-2 and rel(outs[2], outs[0]) < 1e-2


def test_page_split_matches_the_whole_layer():
    """Two and three ranks emulated on one GPU, over steps that fill several pages."""
    from starkv_b200 import context_parallel as cp
    from starkv_b200.full_layer import FullAttentionLayer, FullContextLayer
    w, norms, cs = weights(4, 2, seed=4)
    dev = cs.device
    for world in (2, 3):
        whole = FullAttentionLayer(*w, cs, **norms)
        ranks = [FullContextLayer(*w, cs, rank=r, world=world, **norms) for r in range(world)]
        wc, rc = whole.allocate_cache(9), [r.allocate_cache(9) for r in ranks]
        bt = torch.arange(1, 9, device=dev, dtype=torch.int32).view(2, 4)
        g = torch.Generator(device=dev).manual_seed(8)
        for t in range(55):
            hidden = torch.randn(2, HID, generator=g, device=dev).to(torch.bfloat16)
            pos = torch.full((2,), t, device=dev)
            slots = bt[:, t // 16].long() * 16 + t % 16
            ref = whole.forward(hidden, pos, wc, bt, torch.full((2,), t + 1, dtype=torch.int32, device=dev), 64, slots)
            parts = []
            for r in range(world):
                li = int(cp.local_index(t, world))
                mine = int(cp.page_owner(t, world)) == r
                ls = bt[:, li // 16].long() * 16 + li % 16 if mine else torch.full_like(slots, -1)
                ll = torch.full((2,), int(cp.local_len(t + 1, r, world)), dtype=torch.int32, device=dev)
                parts.append(ranks[r].forward_partial(hidden, pos, rc[r], bt, ll, 64, ls))
            out = F.linear(cp.combine_local(parts).reshape(2, -1), whole.wo)
            assert rel(out, ref) < 1e-2, t


@pytest.mark.parametrize("kw", [dict(), dict(full_top_pages=8), dict(attn_parallel="context")])
def test_model_with_paged_full_layers_matches_dense(kw):
    """The model's decode with this library's full-rank layers against the dense float32
    recomputation that the stock layers are held to, with the same bound."""
    import test_gpu_model as M
    from starkv_b200.model import StarKVModel
    dev = cuda()
    model = StarKVModel(M.small_config(), dev, full_attention="paged", **kw)
    g = torch.Generator(device=dev).manual_seed(1)
    tokens = torch.randint(0, model.cfg.vocab, (M.BATCH, M.STEPS), generator=g, device=dev)
    pages = -(-M.STEPS // 16)
    caches = model.allocate_caches(M.BATCH * pages + 1, M.BATCH * pages + 1)
    bt = torch.arange(M.BATCH * pages, device=dev, dtype=torch.int32).view(M.BATCH, pages) + 1
    for t in range(M.STEPS):
        slots = bt[:, t // 16].long() * 16 + t % 16
        meta = (bt, torch.full((M.BATCH,), t + 1, dtype=torch.int32, device=dev), M.STEPS, slots)
        logits = model.decode_step(tokens[:, t], torch.full((M.BATCH,), t, device=dev), caches, *meta,
                                   local=meta if kw.get("attn_parallel") else None)
    ref = M.dense_reference(model, tokens)
    assert rel(logits, ref) < 3e-2
    assert model.kv_bytes_per_token() > 0


def test_captured_step():
    from starkv_b200.full_layer import FullAttentionLayer
    w, norms, cs = weights(8, 2, seed=6)
    dev = cs.device
    for top in (None, 3):
        layer = FullAttentionLayer(*w, cs, top_pages=top, **norms)
        cache, other = layer.allocate_cache(17), layer.allocate_cache(17)
        bt = torch.arange(1, 17, device=dev, dtype=torch.int32).view(2, 8)
        hidden = torch.zeros(2, HID, dtype=torch.bfloat16, device=dev)
        pos, sl, slots = (torch.zeros(2, dtype=d, device=dev) for d in (torch.int64, torch.int32, torch.int64))
        layer.forward(hidden, pos, other, bt, sl, 128, slots)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer.forward(hidden, pos, cache, bt, sl, 128, slots)
        other = layer.allocate_cache(17)
        for c in cache:
            c.zero_()
        for t in range(100):
            h = torch.randn(2, HID, device=dev).to(torch.bfloat16)
            hidden.copy_(h)
            pos.fill_(t)
            sl.fill_(t + 1)
            slots.copy_(bt[:, t // 16].long() * 16 + t % 16)
            graph.replay()
            want = layer.forward(h, pos.clone(), other, bt, sl.clone(), 128, slots.clone())
            assert torch.equal(out, want), t
