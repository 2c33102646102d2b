"""How exact the paged decode attention is beyond the half step of its output type.

A 16-bit output differs from the nearest one to the float64 value where the computation's
error crosses a rounding border, so the share of such outputs measures that error: it may
not be larger than that of the same formula in elementary f32 operations. Both shares are
counts of rare independent events; 4 square roots of the larger expected count are left
for chance.

bf16 with more than 4 query heads per KV head: the weights keep two parts of 8 bits, which
leave at most 2^-18 of a weight, evenly spread: 2^-18 / sqrt(3) rms, and as much of the
output's own size s in norm, since V has both signs. An output x is not the nearest with
probability |error| / step(x). Outputs are about normal; step(x) = 2^-7 2^k in the binade
[2^k, 2^k+1), each binade below s holds 0.8 2^k / s of the outputs, and the first 12 below s
have steps above the error, so the mean of s / step is 2^7 (12 0.8 + 1), that of |error| is
0.8 2^-18 / sqrt(3) s: 0.8 2^-11 10.6 / sqrt(3) = 2.4e-3 of the outputs on top of f32's.
"""
import pytest
import torch

from test_gpu_paged_attention import check, make, reference, tokens_of

pytestmark = pytest.mark.gpu


def plain(q, K, V, scale, dtype):
    """softmax(scale q K^T) V of one KV head in `dtype`: q [G, D], K and V [T, D]."""
    x = scale * (q.to(dtype) @ K.to(dtype).T)
    w = torch.exp(x - x.amax(-1, keepdim=True))
    return w @ V.to(dtype) / w.sum(-1, keepdim=True)


@pytest.mark.parametrize("lens,H,Hkv,dtype", [([8192] * 12, 32, 32, torch.bfloat16), ([8000] * 12, 64, 8, torch.bfloat16),
                                              ([7001] * 6, 96, 8, torch.bfloat16), ([8191] * 12, 32, 8, torch.float16),
                                              ([8191] * 12, 32, 8, torch.bfloat16), ([6000] * 12, 64, 8, torch.float16)])
def test_outputs_are_the_nearest_as_often_as_with_f32(lens, H, Hkv, dtype):
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make(lens, H, Hkv, dtype=dtype, seed=90 + Hkv, qmag=1.7)
    scale, G = 128 ** -0.5, H // Hkv
    got = paged_attention_decode(q, k, v, bt, sl, max(lens), scale)
    off = off32 = 0
    for b, L in enumerate(lens):
        t = torch.arange(L, device=q.device)
        K, V = tokens_of(k, bt[b], t), tokens_of(v, bt[b], t)
        for h in range(Hkv):
            r = slice(h * G, (h + 1) * G)
            nearest = plain(q[b, r], K[:, h], V[:, h], scale, torch.float64).to(dtype)
            off += int((got[b, r] != nearest).sum())
            off32 += int((plain(q[b, r], K[:, h], V[:, h], scale, torch.float32).to(dtype) != nearest).sum())
    if dtype == torch.bfloat16 and G > 4:
        off32 += 0.8 * 2 ** -11 * 10.6 / 3 ** 0.5 * got.numel()
    assert off <= off32 + 4 * off32 ** 0.5, (off, off32, got.numel())


def exact_partial(q, K, V, scale):
    """(out undivided, m, l) of one KV head in float64."""
    x = scale * (q.double() @ K.double().T)
    m = x.amax(-1)
    w = torch.exp(x - m[:, None])
    return w @ V.double(), m, w.sum(-1)


@pytest.mark.parametrize("H,Hkv,D,dtype,L", [
    (8, 2, 128, torch.bfloat16, 131071), (12, 1, 128, torch.bfloat16, 40001), (17, 1, 128, torch.bfloat16, 9000),
    (40, 1, 64, torch.bfloat16, 20011), (4, 2, 64, torch.bfloat16, 50000), (12, 1, 128, torch.float16, 40001),
    (3, 3, 64, torch.float16, 30001)])
@pytest.mark.parametrize("listed", [False, True])
def test_partial_form_in_norm(H, Hkv, D, dtype, L, listed):
    """Long, rather flat softmax, whole and over every other page, split and joined. The error
    of a head's out and l, in norm: some hundred f32 additions one after another, whose
    roundings add up as a root (10 2^-24), the hardware exponential (2^-22 at most), the
    logits' and the maximum's error (128 products in f32, a few 2^-24 of logits of a few):
    below 2^-20 together. bf16 weights in two parts, or sums that cut off, are above it."""
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    q, k, v, bt, sl = make([L], H, Hkv, D=D, dtype=dtype, seed=H + L)
    scale, G, bs = D ** -0.5, H // Hkv, 16
    P = -(-L // bs)
    pages = torch.arange(0, P, 2, dtype=torch.int32, device=q.device).expand(1, Hkv, -1) if listed else None
    out, m, l = paged_attention_decode(q, k, v, bt, sl, L, scale, pages=pages, return_partial=True)
    t = torch.arange(L, device=q.device)
    if listed:
        t = t[t // bs % 2 == 0]
    K, V = tokens_of(k, bt[0], t), tokens_of(v, bt[0], t)
    for h in range(Hkv):
        r = slice(h * G, (h + 1) * G)
        ro, rm, rl = exact_partial(q[0, r], K[:, h], V[:, h], scale)
        assert ((out[0, r].double() - ro).norm(dim=-1) <= 2.0 ** -20 * ro.norm(dim=-1)).all(), \
            float(((out[0, r].double() - ro).norm(dim=-1) / ro.norm(dim=-1)).max())
        assert ((l[0, r].double() - rl).abs() <= 2.0 ** -20 * rl).all()
        assert ((m[0, r].double() - rm).abs() <= 2.0 ** -20 * rm.abs().clamp(min=1)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hkv,D", [(12, 1, 128), (17, 1, 128), (40, 1, 64), (32, 2, 128), (8, 2, 64), (3, 3, 64)])
@pytest.mark.parametrize("listed", [False, True])
def test_partial_form_at_edge_lengths(H, Hkv, D, dtype, listed):
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    lens = [1, 0, 15, 16, 17, 64, 65, 256, 257, 1003]
    q, k, v, bt, sl = make(lens, H, Hkv, D=D, dtype=dtype, seed=D + H)
    scale, pages = D ** -0.5, None
    if listed:   # any order, a hole among them, 14 pages at most
        g = torch.Generator().manual_seed(H)
        pages = torch.full((len(lens), Hkv, 14), -1, dtype=torch.int32)
        for b, L in enumerate(lens):
            P = -(-L // 16)
            for h in range(Hkv):
                c = min(14, P)
                pages[b, h, :c] = torch.randperm(P, generator=g)[:c].int()
                if c > 3:
                    pages[b, h, 1] = -1
        pages = pages.to(q.device)
    out, m, l = paged_attention_decode(q, k, v, bt, sl, 1003, scale, pages=pages, return_partial=True)
    ref, rm, rl, tol = reference(q, k, v, bt, sl, scale, pages=pages)
    empty = rl == 0
    assert (m[empty] == float("-inf")).all() and (l[empty] == 0).all() and (out[empty] == 0).all()
    assert empty.any() and not empty.all()
    live = ~empty
    assert ((m - rm)[live].abs() <= tol[..., 0][live]).all()
    assert ((l - rl)[live].abs() <= 2 * tol[..., 0][live] * rl[live]).all()
    check((out / l[..., None])[live], ref[live], 2 * tol[live])
