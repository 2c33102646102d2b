"""How exact the paged decode attention is beyond the half step of its output type.

A 16-bit output differs from the nearest one to the float64 value where the computation's
error crosses a rounding border, so the share of such outputs measures that error: it may
not be larger than that of the same formula in elementary f32 operations. Both shares are
counts of rare independent events; 4 square roots of the larger expected count are left
for chance.
"""
import pytest
import torch

from test_gpu_paged_attention import make, tokens_of

pytestmark = pytest.mark.gpu


def plain(q, K, V, scale, dtype):
    """softmax(scale q K^T) V of one KV head in `dtype`: q [G, D], K and V [T, D]."""
    x = scale * (q.to(dtype) @ K.to(dtype).T)
    w = torch.exp(x - x.amax(-1, keepdim=True))
    return w @ V.to(dtype) / w.sum(-1, keepdim=True)


@pytest.mark.parametrize("lens,H,Hkv,dtype", [([8192] * 12, 32, 32, torch.bfloat16), ([8000] * 12, 64, 8, torch.bfloat16),
                                              ([7001] * 6, 96, 8, torch.bfloat16), ([8191] * 12, 32, 8, torch.float16)])
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
    assert off <= off32 + 4 * off32 ** 0.5, (off, off32, got.numel())
