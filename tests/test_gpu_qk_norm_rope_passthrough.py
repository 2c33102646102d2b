"""Channels behind the rotated width are passed through, whatever their neighbours hold:
infinities, NaN, negative zero, in every such channel in turn."""
import pytest
import torch

from test_gpu_qk_norm_rope import cuda, rotary_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,rot", [(128, 64), (128, 48), (64, 16), (128, 112)])
@pytest.mark.parametrize("n", [1, 700])
def test_channels_behind_the_table_stay_as_they_are(D, rot, dtype, n):
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope_write
    dev = cuda()
    g = torch.Generator(device=dev).manual_seed(rot)
    H, Hkv = 7, 3
    qkv = torch.randn(n, H + 2 * Hkv, D, generator=g, device=dev).to(dtype)
    odd = torch.tensor([float("inf"), -float("inf"), float("nan"), -0.0], device=dev).to(dtype)
    row, head = torch.meshgrid(torch.arange(n, device=dev), torch.arange(H + Hkv, device=dev), indexing="ij")
    for k in range(3):   # three odd values a row, among them neighbours at a distance of four
        at = rot + (row * 5 + head + 4 * k) % (D - rot)
        qkv[row, head, at] = odd[(row + head + k) % 4]
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    pos = torch.randint(0, 500, (n,), generator=g, device=dev)
    cs = rotary_table(500, rot, torch.float32, dev)
    kc, vc = (torch.zeros(n // 16 + 1, 16, Hkv, D, dtype=dtype, device=dev) for _ in range(2))
    slots = torch.arange(n, device=dev)
    out = qk_norm_rope_write(q, k, v, pos, cs, kc, vc, slots)
    bits = lambda t: torch.where(t.isnan(), torch.full_like(t, 7.0), t).contiguous().view(torch.int16)   # noqa: E731
    stored = kc.view(-1, Hkv, D)[:n]
    for got, x in ((out, q), (stored, k)):
        assert torch.equal(got.isnan(), x.isnan())
        assert torch.equal(bits(got[..., rot:]), bits(x[..., rot:]))
    assert torch.equal(vc.view(-1, Hkv, D)[:n], v)


def test_normed_channels_behind_the_table():
    """With a norm a row that holds an infinity has mean square infinity: its finite channels
    become 0, the infinite ones NaN, as the formula has it."""
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope
    dev = cuda()
    q = torch.randn(3, 2, 128, device=dev).to(torch.bfloat16)
    q[1, 1, 100] = float("inf")
    w = torch.ones(128, device=dev)
    cs = rotary_table(10, 64, torch.float32, dev)
    out, _ = qk_norm_rope(q, None, torch.zeros(3, dtype=torch.int64, device=dev), cs, q_weight=w)
    assert out[1, 1].isnan().nonzero().tolist() == [[100]]
    assert (out[1, 1, :100] == 0).all() and (out[1, 1, 101:] == 0).all()
    assert torch.isfinite(out[0].float()).all() and torch.isfinite(out[1, 0].float()).all()
