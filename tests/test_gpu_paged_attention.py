"""GPU parity of the full-rank paged decode attention (starkv_paged_attention) against the
formula in float64: out = softmax(scale q K^T) V per sequence and query head.

Tolerance, per element: half a step of the output type (eps / 2 |out|), plus the weights'
errors times the largest |V|. A weight exp(scale q.k - m) / l is off by the logit's error
(head_dim products summed in f32: D 2^-23 scale sum|q k|, in numerator and denominator),
the hardware exponential and the f32 sums (2^-18), and what the two-part weights leave
(2^-16 for bf16). Cache rows that no sequence owns, and rows past a sequence's end, hold
NaN: they must not show.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda", 0)


def make(lens, H, Hkv, D=128, bs=16, dtype=torch.bfloat16, order="head", seed=0, qmag=1.0, table_extra=0):
    """A NaN-filled cache holding the sequences' tokens at random blocks."""
    dev = cuda()
    g = torch.Generator(device=dev).manual_seed(seed)
    n = len(lens)
    per = max(1, -(-max(lens) // bs)) + table_extra
    blocks = n * per + 3
    caches = []
    for _ in range(2):
        if order == "head":
            c = torch.full((blocks, Hkv, bs, D), float("nan"), dtype=dtype, device=dev).transpose(1, 2)
        else:
            c = torch.full((blocks, bs, Hkv, D), float("nan"), dtype=dtype, device=dev)
        caches.append(c)
    perm = torch.randperm(blocks - 1, generator=g, device=dev)[:n * per] + 1
    bt = perm.view(n, per).int()
    for b, L in enumerate(lens):
        t = torch.arange(L, device=dev)
        blk = bt[b, t // bs].long()
        for c in caches:
            c[blk, t % bs] = torch.randn(L, Hkv, D, generator=g, device=dev).to(dtype)
    q = (qmag * torch.randn(n, H, D, generator=g, device=dev)).to(dtype)
    return q, caches[0], caches[1], bt, torch.tensor(lens, dtype=torch.int32, device=dev)


def tokens_of(cache, bt_row, positions):
    bs = cache.shape[1]
    return cache[bt_row[positions // bs].long(), positions % bs]     # [T, Hkv, D]


def reference(q, k_cache, v_cache, bt, lens, scale, pages=None):
    """(out, m, l, tolerance) in float64, out divided."""
    n, H, D = q.shape
    Hkv, bs = k_cache.shape[2], k_cache.shape[1]
    G = H // Hkv
    out = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    m = torch.full((n, H), float("-inf"), dtype=torch.float64, device=q.device)
    l = torch.zeros(n, H, dtype=torch.float64, device=q.device)
    tol = torch.zeros(n, H, 1, dtype=torch.float64, device=q.device)
    for b in range(n):
        L = int(lens[b])
        for h in range(Hkv):
            if pages is None:
                pos = torch.arange(L, device=q.device)
            else:
                listed = pages[b, h][pages[b, h] >= 0].long()
                pos = (listed[:, None] * bs + torch.arange(bs, device=q.device)).reshape(-1)
                pos = pos[pos < L]
            if pos.numel() == 0:
                continue
            K = tokens_of(k_cache, bt[b], pos)[:, h].double()
            V = tokens_of(v_cache, bt[b], pos)[:, h].double()
            Q = q[b, h * G:(h + 1) * G].double()
            x = scale * Q @ K.T
            r = slice(h * G, (h + 1) * G)
            m[b, r] = x.amax(-1)
            w = torch.exp(x - m[b, r, None])
            l[b, r] = w.sum(-1)
            out[b, r] = w @ V / l[b, r, None]
            logit_err = D * 2.0 ** -23 * scale * (Q.abs() @ K.abs().T).amax(-1)
            tol[b, r, 0] = (2 * logit_err + 2.0 ** -16 + 2.0 ** -18) * V.abs().max()
    return out, m, l, tol


def check(got, ref, tol):
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    assert torch.isfinite(got.float()).all()
    assert (err <= half * ref.abs() + tol).all(), float((err - half * ref.abs() - tol).max())


EDGES = [1, 0, 15, 16, 17, 31, 63, 64, 65, 128, 129, 300, 0, 1003]


def run(lens, H, Hkv, D=128, bs=16, dtype=torch.bfloat16, order="head", seed=0, qmag=1.0):
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make(lens, H, Hkv, D, bs, dtype, order, seed, qmag)
    scale = D ** -0.5
    status = torch.zeros(1, dtype=torch.int32, device=q.device)
    out = paged_attention_decode(q, k, v, bt, sl, max(max(lens), 1), scale, status=status)
    assert int(status) == 0
    ref, _, _, tol = reference(q, k, v, bt, sl, scale)
    check(out, ref, tol)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hkv", [(8, 8), (32, 8), (5, 1), (8, 1), (12, 1), (34, 2), (40, 1)])
def test_head_layouts_at_edge_lengths(H, Hkv, dtype):
    # groups of 1, 4, 5, 8 (one half of the MMA rows), 12 (both), 17 and 40 (several row groups)
    run(EDGES, H, Hkv, dtype=dtype, seed=H)


@pytest.mark.parametrize("bs", [1, 5, 16, 24, 32, 48, 64, 256])
@pytest.mark.parametrize("D,order", [(64, "token"), (128, "head"), (128, "token")])
def test_block_sizes_and_orders(bs, D, order):
    run(EDGES, 8, 2, D=D, bs=bs, order=order, seed=bs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_long_sequence_is_split_and_joined(dtype):
    run([40001], 8, 2, dtype=dtype, seed=1)


@pytest.mark.parametrize("H,Hkv,lens", [(8, 8, [2500, 1300]), (5, 1, [12000, 9001]), (6, 2, [3000, 5000, 70]),
                                        (12, 1, [9000, 9000, 9000]), (17, 1, [7000, 4000])])
@pytest.mark.parametrize("D", [64, 128])
def test_shares_that_end_one_unit_and_begin_another(H, Hkv, lens, D):
    # several tiles per share, so that both partial slots of a share are in use, for odd and even groups
    run(lens, H, Hkv, D=D, seed=H)


def test_many_sequences():
    # more sequences than a warp looks at in one step, most of them short
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 90, (301,), generator=g).tolist()
    lens[7], lens[200] = 2500, 1777
    run(lens, 4, 2, seed=2)


def test_peaked_and_flat_weights():
    run([700, 9, 2100], 8, 2, qmag=8.0, seed=3)
    run([700, 9, 2100], 8, 2, qmag=0.0, seed=4)
    run([5000], 4, 1, dtype=torch.float16, qmag=6.0, seed=5)


def test_same_bits_every_time():
    a = run([4096, 100, 2222], 8, 2, seed=6)
    assert torch.equal(a, run([4096, 100, 2222], 8, 2, seed=6))


def test_longer_than_max_seq_len_is_cut():
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make([100, 300], 4, 2)
    out = paged_attention_decode(q, k, v, bt, sl, 130, 0.1)
    ref, _, _, tol = reference(q, k, v, bt, sl.clamp(max=130), 0.1)
    check(out, ref, tol)


def test_strided_tensors():
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make([70, 513, 5], 8, 2)
    fused = torch.randn(3, 24, 128, device=q.device).to(q.dtype)
    fused[:, 4:12] = q
    both = torch.randn(3, 2, 8, 128, device=q.device).to(q.dtype)
    keep = both.clone()
    wide = torch.zeros(bt.shape[1], 6, dtype=torch.int32, device=q.device)
    wide[:, ::2] = bt.T
    out = paged_attention_decode(fused[:, 4:12], k, v, wide[:, ::2].T, sl, 513, 0.1, out=both[:, 1])
    assert out.data_ptr() == both[:, 1].data_ptr()
    ref, _, _, tol = reference(q, k, v, bt, sl, 0.1)
    check(out, ref, tol)
    assert torch.equal(both[:, 0], keep[:, 0])
    # int64 lengths and tables are taken too
    again = paged_attention_decode(q, k, v, bt.long(), sl.long(), 513, 0.1)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 128), (torch.float16, 64)])
def test_partial_form(dtype, D):
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make([2000, 0, 33], 8, 2, D=D, dtype=dtype, seed=7)
    scale = D ** -0.5
    out, m, l = paged_attention_decode(q, k, v, bt, sl, 2000, scale, return_partial=True)
    ref, rm, rl, tol = reference(q, k, v, bt, sl, scale)
    assert out.dtype == m.dtype == l.dtype == torch.float32
    assert torch.equal(m[1], torch.full_like(m[1], float("-inf"))) and (l[1] == 0).all() and (out[1] == 0).all()
    rows = [0, 2]
    assert ((m - rm)[rows].abs() <= tol[rows, :, 0]).all()     # tol bounds the logits' error, |V| > 1
    assert ((l - rl)[rows].abs() <= 2 * tol[rows, :, 0] * rl[rows]).all()
    check((out / l[..., None])[rows], ref[rows], 2 * tol[rows])


def test_partials_of_a_page_split_combine_to_the_whole():
    from starkv_b200.context_parallel import combine_local
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make([1000, 40, 7], 8, 8, seed=8)
    parts = []
    for r in range(3):
        mine = bt[:, r::3].contiguous()
        full, rest = sl // 16, sl % 16          # rank r holds pages r, r + 3, ...
        local = ((full - r + 2).clamp(min=0) // 3) * 16 + torch.where(full % 3 == r, rest, 0)
        parts.append(paged_attention_decode(q, k, v, mine, local, 1000, 0.09, return_partial=True))
    out = combine_local(parts)
    ref, _, _, tol = reference(q, k, v, bt, sl, 0.09)
    check(out, ref, 2 * tol)


def test_blocks_outside_the_cache_are_recorded():
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make([100, 40], 4, 2)
    k[0], v[0] = 0, 0                            # what a bad block id reads instead
    bt[0, 2], bt[1, 1] = 10 ** 6, -1
    status = torch.zeros(1, dtype=torch.int32, device=q.device)
    out = paged_attention_decode(q, k, v, bt, sl, 100, 0.1, status=status)
    assert int(status) == 105
    bt[0, 2] = bt[1, 1] = 0
    ref, _, _, tol = reference(q, k, v, bt, sl, 0.1)
    check(out, ref, tol)


def test_stream_and_graphs():
    """Another stream; a captured call replayed with other lengths; two graphs at once."""
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    cases = [make([900, 64, 1], 8, 2, seed=20), make([5, 1500, 333], 8, 2, seed=21)]
    outs, graphs, side = [], [], torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in cases:
            paged_attention_decode(*c, 1500, 0.1)
    torch.cuda.synchronize()
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(paged_attention_decode(*c, 1500, 0.1))
        graphs.append(g)
    cases[0][4].copy_(torch.tensor([17, 64, 800], dtype=torch.int32))   # within the first one's blocks
    q, k, v, bt, sl = cases[0]
    t = torch.arange(800, device=q.device)
    k[bt[2, t // 16].long(), t % 16] = torch.randn(800, 2, 128, device=q.device).to(k.dtype)
    v[bt[2, t // 16].long(), t % 16] = torch.randn(800, 2, 128, device=q.device).to(v.dtype)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, out in zip(cases, outs):
        ref, _, _, tol = reference(*c, 0.1)
        check(out, ref, tol)


def test_empty_batch():
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make([3], 4, 2)
    out = paged_attention_decode(q[:0], k, v, bt[:0], sl[:0], 3, 0.1)
    assert out.shape == (0, 4, 128)


@pytest.mark.parametrize("H,Hkv,bs,D", [(8, 2, 16, 128), (12, 1, 24, 128), (4, 4, 5, 64), (8, 1, 64, 64)])
def test_listed_pages(H, Hkv, bs, D):
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    lens = [0, 1, 7 * bs, 20 * bs + 3, 40 * bs - 1]
    q, k, v, bt, sl = make(lens, H, Hkv, D=D, bs=bs, seed=bs)
    g = torch.Generator().manual_seed(1)
    pages = torch.full((5, Hkv, 9), -1, dtype=torch.int32)
    for b, L in enumerate(lens):
        P = -(-L // bs)
        for h in range(Hkv):
            c = min(9, P)
            pages[b, h, :c] = torch.randperm(P, generator=g)[:c].int()     # any order
            if c > 4:
                pages[b, h, 2] = -1                                         # a hole
            if c > 5:
                pages[b, h, 4] = 10 ** 6                                    # past the sequence: no token
    dev_pages = pages.to(q.device)
    status = torch.zeros(1, dtype=torch.int32, device=q.device)
    out = paged_attention_decode(q, k, v, bt, sl, 41 * bs, 0.1, pages=dev_pages, status=status)
    assert int(status) == 0
    ref, _, _, tol = reference(q, k, v, bt, sl, 0.1, pages=torch.where(pages == 10 ** 6, -1, pages).to(q.device))
    check(out, ref, tol)


def test_a_page_listed_twice_counts_twice():
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make([64], 2, 1)
    two = torch.tensor([[[1, 3, 1]]], dtype=torch.int32, device=q.device)
    out = paged_attention_decode(q, k, v, bt, sl, 64, 0.1, pages=two)
    ref, _, _, tol = reference(q, k, v, bt, sl, 0.1, pages=two)
    check(out, ref, tol)


def test_cache_of_more_than_two_to_the_31_elements():
    """Blocks at the far end of a cache whose offsets pass 32 bits, keys and values as views of
    one tensor [blocks, 2, heads, block, 128]."""
    from starkv_b200.kernels.paged_attention import empty_bounds, paged_attention_decode, sparse_paged_decode, \
        update_page_bounds
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope_write
    dev = cuda()
    if torch.cuda.mem_get_info(dev)[0] < 8 << 30:
        pytest.skip("needs 8 GB")
    Hkv, bs, n, T = 8, 16, 2, 300
    blocks = (1 << 31) // (2 * Hkv * bs * 128) + 64
    both = torch.empty(blocks, 2, Hkv, bs, 128, dtype=torch.bfloat16, device=dev)
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    assert (blocks - 1) * k.stride(0) > 1 << 31
    per = -(-T // bs)
    bt = (blocks - 1 - torch.arange(n * per, device=dev).view(n, per)).int()
    qkv = torch.randn(n * T, 32 + 2 * Hkv, 128, device=dev).to(torch.bfloat16)
    t = torch.arange(T, device=dev)
    slots = (bt[:, t // bs].long() * bs + t % bs).reshape(-1)
    cs = torch.cat([torch.ones(8, 64, device=dev), torch.zeros(8, 64, device=dev)], 1)     # no rotation
    qk = qk_norm_rope_write(qkv[:, :32], qkv[:, 32:40], qkv[:, 40:], torch.zeros(n * T, dtype=torch.int64, device=dev), cs,
                            k, v, slots)
    assert torch.equal(qk, qkv[:, :32])
    assert torch.equal(tokens_of(k, bt[1], t), qkv[T:, 32:40]) and torch.equal(tokens_of(v, bt[0], t), qkv[:T, 40:])
    sl = torch.tensor([T, T - 9], dtype=torch.int32, device=dev)
    q = qk[:2]
    ref, _, _, tol = reference(q, k, v, bt, sl, 0.1)
    check(paged_attention_decode(q, k, v, bt, sl, T, 0.1), ref, tol)
    bounds = empty_bounds(k)
    update_page_bounds(k, bounds, bt, sl, T, max_new=T)
    out, pages = sparse_paged_decode(q, k, v, bounds, bt, sl, T, 0.1, 5)
    ref, _, _, tol = reference(q, k, v, bt, sl, 0.1, pages=pages)
    check(out, ref, tol)


def test_shared_heads_of_an_expanded_cache():
    """A cache whose head stride is 0 (one stored head seen as four)."""
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make([400, 3], 8, 1, seed=31)
    k4, v4 = k.expand(-1, -1, 4, -1), v.expand(-1, -1, 4, -1)
    out = paged_attention_decode(q, k4, v4, bt, sl, 400, 0.1)
    ref, _, _, tol = reference(q, k, v, bt, sl, 0.1)
    check(out, ref, tol)


def test_own_workspace():
    from starkv_b200.kernels.paged_attention import paged_attention_decode, workspace_bytes
    q, k, v, bt, sl = make([5000, 200], 8, 2, seed=32)
    ws = torch.empty(workspace_bytes(8, 2, 128, 5000), dtype=torch.uint8, device=q.device)
    a = paged_attention_decode(q, k, v, bt, sl, 5000, 0.1, ws=ws)
    assert torch.equal(a, paged_attention_decode(q, k, v, bt, sl, 5000, 0.1))
    with pytest.raises(RuntimeError, match="workspace"):
        paged_attention_decode(q, k, v, bt, sl, 5000, 0.1, ws=ws[:-16])
