"""Infinite and NaN values in V: a channel that holds an infinity is that infinity (every
weight is above 0), NaN where both signs or a NaN meet, and no other channel, head or
sequence shows any of it."""
import pytest
import torch

from test_gpu_paged_attention import check, make, reference

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def spoil(k, v, bt, b, L, q, h, G, bs):
    """Infinities and NaN in KV head h of sequence b: {channel: what its outputs are}. The odd
    tokens are the one of the largest weight, the one of the smallest, and the last one."""
    t = torch.arange(L, device=v.device)
    blk, off = bt[b, t // bs].long(), t % bs
    logit = k[blk, off, h].double() @ q[b, h * G].double()
    peak, least, last = int(logit.argmax()), int(logit.argmin()), L - 1

    def put(tok, c, x):
        v[bt[b, tok // bs].long(), tok % bs, h, c] = x
    put(peak, 0, INF)
    put(peak, 3, -INF)
    put(least, 8, INF)
    put(least, 13, -INF)
    put(last, 17, -INF)
    put(peak, 21, INF)
    put(least, 21, INF)
    put(peak, 26, INF)
    put(last if last != peak else least, 26, -INF)
    put(last, 63, NAN)
    return {0: INF, 3: -INF, 8: INF, 13: -INF, 17: -INF, 21: INF, 26: NAN, 63: NAN}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hkv,D,bs", [(4, 4, 128, 16), (8, 2, 128, 16), (12, 1, 128, 24), (40, 2, 64, 16), (5, 1, 64, 5)])
@pytest.mark.parametrize("form", ["dense", "partial", "pages"])
def test_values_that_are_not_finite(H, Hkv, D, bs, dtype, form):
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    lens = [40, 200, 3000, 7777]                     # whole units, and units over many shares
    q, k, v, bt, sl = make(lens, H, Hkv, D=D, bs=bs, dtype=dtype, seed=H + D, qmag=3.0)
    clean = v.clone()
    G, h = H // Hkv, Hkv - 1
    pages = None
    if form == "pages":                              # every page listed, so the odd tokens are among them
        P = -(-max(lens) // bs)
        pages = torch.arange(P, dtype=torch.int32, device=q.device).expand(4, Hkv, P)
        pages = torch.where(pages < ((sl + bs - 1) // bs)[:, None, None], pages, -1)
    want = [spoil(k, v, bt, b, L, q, h, G, bs) for b, L in enumerate(lens) if b != 1]
    want.insert(1, {})
    scale = D ** -0.5
    out = paged_attention_decode(q, k, v, bt, sl, max(lens), scale, pages=pages, return_partial=form == "partial")
    if form == "partial":
        out, _, l = out
        assert torch.isfinite(l).all()
        out = out / l[..., None]
    ref, _, _, tol = reference(q, k, clean, bt, sl, scale)
    odd = torch.zeros(out.shape, dtype=torch.bool, device=out.device)
    for b, w in enumerate(want):
        for c, x in w.items():
            odd[b, h * G:, c] = True
            got = out[b, h * G:, c].float()
            assert (got.isnan() if x != x else got == x).all(), (b, c, x, got)
    check(torch.where(odd, ref.to(out.dtype), out), ref, 2 * tol)


def test_infinity_where_the_weights_underflow():
    """Logits so far apart that the weight of the infinite token is 0 in f32, in one share and
    between shares."""
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    for L in (100, 5000):
        q, k, v, bt, sl = make([L], 2, 1, seed=L)
        q.zero_()
        q[..., 0] = 1
        t = torch.arange(L, device=q.device)
        k[bt[0, t // 16].long(), t % 16] = 0
        k[bt[0, 1].long(), 3, 0, 0] = 300            # token 19; the others' weights are e^-300
        v[bt[0, (L - 1) // 16].long(), (L - 1) % 16, 0, 5] = -INF
        out = paged_attention_decode(q, k, v, bt, sl, L, 1.0)
        assert (out[..., 5] == -INF).all()
        other = [c for c in range(128) if c != 5]
        assert torch.equal(out[0, 0, other], v[bt[0, 1].long(), 3, 0, other])


def test_queries_that_are_not_finite_stay_their_own():
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make([3000, 50], 8, 2, seed=3)
    ref, _, _, tol = reference(q, k, v, bt, sl, 0.1)
    q[0, 5, 7] = NAN
    q[1, 1, 0] = INF                                 # logits of both infinities: NaN
    out = paged_attention_decode(q, k, v, bt, sl, 3000, 0.1)
    assert out[0, 5].isnan().all() and out[1, 1].isnan().all()
    out[0, 5], out[1, 1] = ref[0, 5].to(out.dtype), ref[1, 1].to(out.dtype)
    check(out, ref, tol)
