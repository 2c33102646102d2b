"""GPU checks of the page bounds (exact: smallest and largest value) and of the page
selection, whose result is compared as whole numbers with a float64 sort of
sum_{g, d} max(q lo, q hi), ties to the lowest page."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda", 0)


def table(n, per, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randperm(n * per, generator=g) + 1).view(n, per).int().to(cuda())


def expected(q, bounds, bt, lens, bs, top, sinks, recent):
    n, H, D = q.shape
    Hkv = bounds.shape[1]
    G = H // Hkv
    out = torch.full((n, Hkv, top), -1, dtype=torch.int32)
    for b in range(n):
        P = -(-int(lens[b]) // bs)
        for h in range(Hkv):
            if P <= top:
                out[b, h, :P] = torch.arange(P)
                continue
            B = bounds[bt[b, :P].long(), h].double()
            Q = q[b, h * G:(h + 1) * G].double()
            s = torch.maximum(Q[:, None] * B[:, 0], Q[:, None] * B[:, 1]).sum((0, 2))
            s = torch.where(s.isnan(), float("inf"), s)
            keep = list(range(sinks)) + list(range(P - recent, P))
            kept = set(keep)
            rest = [i for i in torch.argsort(s, descending=True, stable=True).tolist() if i not in kept]
            out[b, h] = torch.tensor(sorted(keep + rest[:top - len(keep)]), dtype=torch.int32)
    return out


def run(lens, H, Hkv, D=128, bs=16, top=8, sinks=1, recent=1, dtype=torch.bfloat16, seed=0, levels=None, zero_q=False):
    from starkv_b200.kernels.paged_attention import select_pages
    dev = cuda()
    g = torch.Generator(device=dev).manual_seed(seed)
    n, per = len(lens), max(1, -(-max(lens) // bs))
    bt = table(n, per, seed)
    a, c = (torch.randn(n * per + 1, Hkv, D, generator=g, device=dev) for _ in range(2))
    if levels:    # few distinct values: many equal scores
        a, c = (a * levels).round() / levels, (c * levels).round() / levels
    bounds = torch.stack([torch.minimum(a, c), torch.maximum(a, c)], 2).to(dtype)
    q = torch.randn(n, H, D, generator=g, device=dev).to(dtype)
    if levels:
        q = (q * levels).round() / levels
    if zero_q:
        q.zero_()
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    got = select_pages(q, bounds, bt, sl, max(max(lens), 1), bs, top, sinks=sinks, recent=recent, status=status)
    assert int(status) == 0
    assert torch.equal(got.cpu(), expected(q, bounds, bt, lens, bs, top, sinks, recent))


LENS = [0, 1, 16, 17, 127, 128, 129, 145, 1000, 5000]


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 128), (torch.bfloat16, 64)])
@pytest.mark.parametrize("H,Hkv", [(4, 4), (8, 2), (5, 1), (6, 3), (11, 11), (40, 20)])
def test_selection_at_edge_lengths(H, Hkv, dtype, D):
    run(LENS, H, Hkv, D=D, dtype=dtype, seed=H)


@pytest.mark.parametrize("top,sinks,recent", [(1, 0, 0), (1, 0, 1), (2, 1, 1), (9, 4, 3), (33, 0, 0), (300, 1, 1)])
def test_kept_pages(top, sinks, recent):
    run(LENS, 8, 2, top=top, sinks=sinks, recent=recent, seed=top)


@pytest.mark.parametrize("bs", [1, 5, 16, 64])
def test_block_sizes(bs):
    run([3 * bs, 40 * bs + 1, 333], 4, 2, bs=bs, seed=bs)


def test_long_sequences_over_a_cluster():
    run([131071], 8, 2, top=64, seed=1)
    run([70000, 12, 30000], 4, 1, top=129, seed=2)


def test_ties_go_to_the_lowest_page():
    run([16 * 700], 4, 2, top=50, levels=1, D=64, seed=3)
    run([16 * 5000, 16 * 300], 4, 1, top=77, zero_q=True, seed=4)     # all scores equal
    run([16 * 700] * 40, 4, 4, top=10, levels=1, D=64, seed=5)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_scores_that_32_bits_cannot_tell_apart(dtype, D):
    """A common part of 256 (its last place in f32: 2^-15) and differences of multiples of
    2^-20: the order is only there in 64 bits. Some pages stand clearly above and below."""
    from starkv_b200.kernels.paged_attention import select_pages
    dev = cuda()
    g = torch.Generator(device=dev).manual_seed(11)
    n, P, Hkv = 3, 900, 2
    bt = table(n, P, 1)
    b = torch.zeros(n * P + 1, Hkv, D, device=dev)
    b[..., 0] = 16
    j = torch.randint(0, 200, b.shape[:2], generator=g, device=dev)
    b[..., 1] = j * 2.0 ** -16                            # bf16 and f16 hold them
    far = torch.rand(b.shape[:2], generator=g, device=dev)
    b[..., 2] = torch.where(far < 0.01, 1.0, torch.where(far > 0.9, -1.0, 0.0))
    bounds = torch.stack([b, b], 2).to(dtype)
    assert torch.equal(bounds[:, :, 0].float(), b)
    q = torch.zeros(n, 4, D, device=dev)
    q[:, ::2, 0], q[:, ::2, 1], q[:, ::2, 2] = 16, 2.0 ** -4, 1
    q = q.to(dtype)
    sl = torch.tensor([16 * P, 16 * 70, 16 * 400], dtype=torch.int32, device=dev)
    for top in (40, 65):
        got = select_pages(q, bounds, bt, sl, 16 * P, 16, top)
        assert torch.equal(got.cpu(), expected(q, bounds, bt, sl.tolist(), 16, top, 1, 1))


def test_infinite_bounds():
    from starkv_b200.kernels.paged_attention import select_pages
    dev = cuda()
    bounds = torch.randn(301, 1, 2, 128, device=dev).sort(2).values.to(torch.bfloat16)
    bounds[50, 0, 1, 3] = bounds[200, 0, 1, 3] = float("inf")
    bounds[90, 0, 0, 3] = bounds[91, 0, 1, 4] = float("-inf")
    bt = torch.arange(1, 301, device=dev, dtype=torch.int32)[None]
    q = torch.randn(1, 2, 128, device=dev).abs().to(torch.bfloat16)
    q[:, 0, 7] = -1
    sl = torch.tensor([4800], dtype=torch.int32, device=dev)
    for top in (1, 2, 30, 298, 299):
        got = select_pages(q, bounds, bt, sl, 4800, 16, top, sinks=0, recent=0)
        up, down = q.double().clamp(min=0).sum(1), q.double().clamp(max=0).sum(1)
        B = bounds[1:, 0].double()
        s = (up * B[:, 1] + down * B[:, 0]).sum(-1)       # 0 times an infinity: NaN, which ranks first
        s = torch.where(s.isnan(), float("inf"), s) + torch.where(s.isnan(), 1.0, 0.0)
        nan = (up * B[:, 1] + down * B[:, 0]).sum(-1).isnan()
        order = sorted(range(300), key=lambda i: (not bool(nan[i]), -float(s[i]), i))[:top]
        assert got[0, 0].tolist() == sorted(order), top


def test_nan_bounds_rank_first():
    from starkv_b200.kernels.paged_attention import select_pages
    dev = cuda()
    bounds = torch.randn(101, 1, 2, 128, device=dev).sort(2).values.to(torch.bfloat16)
    bt = torch.arange(1, 101, device=dev, dtype=torch.int32)[None]
    bounds[41, 0, 0, 5] = float("nan")
    bounds[73, 0, 1, 9] = -float("nan")
    q = torch.randn(1, 2, 128, device=dev).to(torch.bfloat16)
    got = select_pages(q, bounds, bt, torch.tensor([1600], dtype=torch.int32, device=dev), 1600, 16, 2, sinks=0,
                       recent=0)
    assert got.tolist() == [[[40, 72]]]


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("bs", [1, 5, 16, 64])
@pytest.mark.parametrize("order", ["head", "token"])
def test_bounds(dtype, D, bs, order):
    from starkv_b200.kernels.paged_attention import empty_bounds, update_page_bounds
    dev = cuda()
    g = torch.Generator(device=dev).manual_seed(bs)
    lens = torch.tensor([0, 1, bs, bs + 1, 5 * bs - 1, 200])
    Hkv, n = 3, len(lens)
    per = -(-int(lens.max()) // bs)
    bt = table(n, per, 3)
    shape = (n * per + 1, Hkv, bs, D)
    k = torch.randn(shape, generator=g, device=dev).to(dtype)
    k = k.transpose(1, 2) if order == "head" else k.transpose(1, 2).contiguous()
    sl = lens.int().to(dev)
    k[bt[5, 0].long(), 0, 1, 7] = float("nan")
    k[bt[5, 1].long(), 0, 2, 3] = float("-inf")
    for new in (1, 3, 1000, None):
        new_lens = None if new is not None else torch.tensor([4, 0, 2, bs, 1, 150], dtype=torch.int32, device=dev)
        bounds = empty_bounds(k)
        bounds.fill_(9.0)
        want = bounds.clone()
        for b, L in enumerate(lens.tolist()):
            fresh = min(L, new if new is not None else int(new_lens[b]))
            for p in range((L - fresh) // bs, -(-L // bs)) if fresh else []:
                rows = k[bt[b, p].long(), :min(bs, L - p * bs)]
                want[bt[b, p].long(), :, 0], want[bt[b, p].long(), :, 1] = rows.amin(0), rows.amax(0)
        update_page_bounds(k, bounds, bt, sl, int(lens.max()), max_new=new or 150, new_lens=new_lens)
        same = torch.equal(torch.nan_to_num(bounds, nan=77.0), torch.nan_to_num(want, nan=77.0))
        assert same, new


def test_bounds_record_blocks_outside_the_cache():
    from starkv_b200.kernels.paged_attention import empty_bounds, select_pages, update_page_bounds
    dev = cuda()
    k = torch.randn(5, 16, 1, 128, device=dev).to(torch.bfloat16)
    bt = torch.tensor([[1, 99, 3, 4]], dtype=torch.int32, device=dev)
    sl = torch.tensor([60], dtype=torch.int32, device=dev)
    bounds = empty_bounds(k)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    update_page_bounds(k, bounds, bt, sl, 64, max_new=60, status=status)
    assert int(status) == 105 and (bounds[2] == 0).all()
    q = torch.randn(1, 1, 128, device=dev).to(torch.bfloat16)
    status.zero_()
    select_pages(q, bounds, bt, sl, 64, 16, 2, sinks=0, recent=0, status=status)
    assert int(status) == 105


def test_sparse_decode_is_the_attention_over_the_selected_pages():
    """The whole path of a step: bounds kept page by page while a sequence grows, selection,
    attention; with enough pages it is the full attention."""
    import test_gpu_paged_attention as A
    from starkv_b200.kernels.paged_attention import (empty_bounds, paged_attention_decode, sparse_paged_decode,
                                                     update_page_bounds)
    q, k, v, bt, sl = A.make([1000, 0, 333, 2047], 8, 2, seed=30)
    bounds = empty_bounds(k)
    update_page_bounds(k, bounds, bt, sl, 2047, max_new=2047)
    out, pages = sparse_paged_decode(q, k, v, bounds, bt, sl, 2047, 0.1, 12)
    assert torch.equal(pages.cpu(), expected(q, bounds, bt, sl.tolist(), 16, 12, 1, 1))
    ref, _, _, tol = A.reference(q, k, v, bt, sl, 0.1, pages=pages)
    A.check(out, ref, tol)
    all_pages, _ = sparse_paged_decode(q, k, v, bounds, bt, sl, 2047, 0.1, 128)
    assert torch.equal(all_pages, paged_attention_decode(q, k, v, bt, sl, 2047, 0.1))
    # captured and replayed
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        again, _ = sparse_paged_decode(q, k, v, bounds, bt, sl, 2047, 0.1, 12)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, out)


@pytest.mark.parametrize("P,n", [(200, 2), (500, 2), (900, 2), (2100, 2), (9100, 2), (40, 80), (900, 80)])
@pytest.mark.parametrize("kind", ["equal", "few values", "spread", "nan"])
def test_every_way_to_the_border(P, n, kind):
    """Few and many pages next to the border, equal pages, NaN among them; units that are
    scored in one kernel with the selection (few, up to 512 pages) and in two (long ones,
    also longer than what is copied to shared memory, and more units than SMs)."""
    from starkv_b200.kernels.paged_attention import select_pages
    dev = cuda()
    g = torch.Generator(device=dev).manual_seed(P)
    a, c = (torch.randn(P + 1, 2, 64, generator=g, device=dev) for _ in range(2))
    if kind == "equal":
        a[:], c[:] = a[0].clone(), c[0].clone()
    if kind == "few values":
        pick = torch.randint(0, 3, (P + 1,), generator=g, device=dev)
        a, c = a[:3][pick], c[:3][pick]
    bounds = torch.stack([torch.minimum(a, c), torch.maximum(a, c)], 2).to(torch.bfloat16)
    if kind == "nan":
        bounds[torch.randint(1, P, (40,), generator=g, device=dev), 1, 0, 3] = float("nan")
    q = torch.randn(n, 6, 64, generator=g, device=dev).to(torch.bfloat16)
    bt = torch.arange(1, P + 1, device=dev, dtype=torch.int32).expand(n, P)      # one table row for all
    sl = torch.tensor([P, P - 7] * (n // 2), dtype=torch.int32, device=dev)
    for top in (2, 30, 170):
        got = select_pages(q, bounds, bt, sl, P, 1, top)
        assert torch.equal(got.cpu(), expected(q, bounds, bt, sl.tolist(), 1, top, 1, 1)), top


def test_two_selections_at_once():
    from starkv_b200.kernels.paged_attention import sparse_paged_decode
    import test_gpu_paged_attention as A
    from starkv_b200.kernels.paged_attention import empty_bounds, update_page_bounds
    graphs, outs, args = [], [], []
    for seed, lens in ((40, [3000, 17, 900]), (41, [5, 2000, 2500])):
        q, k, v, bt, sl = A.make(lens, 8, 2, seed=seed)
        b = empty_bounds(k)
        update_page_bounds(k, b, bt, sl, 3000, max_new=3000)
        sparse_paged_decode(q, k, v, b, bt, sl, 3000, 0.1, 9)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(sparse_paged_decode(q, k, v, b, bt, sl, 3000, 0.1, 9))
        args.append((q, k, v, b, bt, sl))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (q, k, v, b, bt, sl), (out, pages) in zip(args, outs):
        assert torch.equal(pages.cpu(), expected(q, b, bt, sl.tolist(), 16, 9, 1, 1))
        ref, _, _, tol = A.reference(q, k, v, bt, sl, 0.1, pages=pages)
        A.check(out, ref, tol)


def test_given_outputs_strided_bounds_and_empty_batches():
    from starkv_b200.kernels.paged_attention import select_pages, sparse_paged_decode, update_page_bounds
    import test_gpu_paged_attention as A
    q, k, v, bt, sl = A.make([900, 20], 4, 2, seed=50)
    wide = torch.full((k.shape[0], 3, 2, 128), 5.0, dtype=k.dtype, device=k.device)
    bounds = wide[:, :2]
    update_page_bounds(k, bounds, bt.long(), sl.long(), 900, max_new=900)
    assert (wide[:, 2] == 5).all()
    both = torch.full((2, 2, 2, 7), -9, dtype=torch.int32, device=k.device)
    lens = torch.stack([sl, sl + 1], 1)[:, 0]                   # a strided view
    got = select_pages(q, bounds, bt, lens, 900, 16, 7, out=both[:, 1])
    assert got.data_ptr() == both[:, 1].data_ptr() and (both[:, 0] == -9).all()
    assert torch.equal(got.cpu(), expected(q, bounds, bt, sl.tolist(), 16, 7, 1, 1))
    out, pages = sparse_paged_decode(q, k, v, bounds, bt, lens, 900, 0.1, 7)
    assert torch.equal(pages, got)
    ref, _, _, tol = A.reference(q, k, v, bt, sl, 0.1, pages=pages)
    A.check(out, ref, tol)
    assert select_pages(q[:0], bounds, bt[:0], sl[:0], 900, 16, 7).shape == (0, 2, 7)
    out, pages = sparse_paged_decode(q[:0], k, v, bounds, bt[:0], sl[:0], 900, 0.1, 7)
    assert out.shape == (0, 4, 128) and pages.shape == (0, 2, 7)
    before = wide.clone()
    update_page_bounds(k, bounds, bt[:0], sl[:0], 900)
    update_page_bounds(k, bounds, bt, sl, 900, max_new=0)
    assert torch.equal(wide, before)


@pytest.mark.parametrize("Hkv,D", [(1, 128), (3, 64), (8, 128), (11, 64), (20, 128)])
@pytest.mark.parametrize("apart", [False, True])
def test_long_units_of_neighbouring_heads(Hkv, D, apart):
    """More pages than one kernel takes; the bounds of a page's heads in one piece, or apart."""
    from starkv_b200.kernels.paged_attention import empty_bounds, select_pages, update_page_bounds
    import test_gpu_paged_attention as A
    q, k, v, bt, sl = A.make([8999, 20, 9600], 2 * Hkv, Hkv, D=D, seed=70 + Hkv)
    bounds = empty_bounds(k)
    if apart:
        bounds = torch.full((k.shape[0], Hkv, 4, D), 7.0, dtype=k.dtype, device=k.device)[:, :, 1:3]
    update_page_bounds(k, bounds, bt, sl, 9600, max_new=9600)
    got = select_pages(q, bounds, bt, sl, 9600, 16, 37)
    assert torch.equal(got.cpu(), expected(q, bounds, bt, sl.tolist(), 16, 37, 1, 1))
