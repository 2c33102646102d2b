"""The selection after a wait of its scoring kernel has run out: the status word says so, the
lists of the units without scores hold -1, nothing else is written, and the workspace's old
contents (here arbitrary bytes) decide nothing."""
import pytest
import torch

from test_gpu_select_pages import cuda, expected, table

pytestmark = pytest.mark.gpu


def test_lists_of_minus_one_after_an_expired_wait():
    from starkv_b200 import _lib
    from starkv_b200.kernels.paged_attention import (empty_cache, paged_attention_decode, select_pages,
                                                     select_workspace_bytes)
    Hkv, D = 11, 64                  # two groups of heads abreast, the second not full
    dev = cuda()
    g = torch.Generator(device=dev).manual_seed(D)
    lens, bs, top = [9600, 7 * 16, 9000, 0], 16, 20
    n, per = len(lens), 600
    bt, sl = table(n, per), torch.tensor(lens, dtype=torch.int32, device=dev)
    bounds = torch.randn(n * per + 1, Hkv, 2, D, generator=g, device=dev).sort(2).values.bfloat16()
    q = torch.randn(n, 2 * Hkv, D, generator=g, device=dev).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = torch.randint(0, 256, (select_workspace_bytes(n, Hkv, 9600, bs, top),), generator=g, device=dev,
                       dtype=torch.uint8)
    both = torch.full((n, Hkv, 2, top), -9, dtype=torch.int32, device=dev)
    out = both[:, :, 1]
    a = _lib.pack_select_pages(
        q.data_ptr(), *q.stride()[:2], bounds.data_ptr(), *bounds.stride()[:2], bt.data_ptr(), *bt.stride(),
        sl.data_ptr(), out.data_ptr(), *out.stride()[:2], status.data_ptr(), _lib.BF16, n, 2 * Hkv, Hkv, D,
        n * per + 1, bs, per, 9600, top, 1, 1)
    _lib.check(_lib.lib().starkv_selftest_select_timeout(a, ws.data_ptr(), ws.nbytes, _lib.stream_ptr(dev)), "selftest")
    torch.cuda.synchronize()
    assert int(status) == 106
    assert (both[:, :, 0] == -9).all()
    assert (out[0] == -1).all() and (out[2] == -1).all() and (out[3] == -1).all()
    assert (out[1] == torch.tensor([*range(7)] + [-1] * 13, device=dev)).all()     # nothing to choose there
    # the attention over such lists is that over no tokens
    k, v = empty_cache(n * per + 1, bs, Hkv, D)
    k.normal_()
    v.normal_()
    attn = paged_attention_decode(q, k, v, bt, sl, 9600, 0.1, pages=out)
    assert (attn[[0, 2, 3]] == 0).all() and (attn[1] != 0).any()
    # and the next call is as ever
    status.zero_()
    got = select_pages(q, bounds, bt, sl, 9600, bs, top, ws=ws, status=status)
    assert int(status) == 0
    assert torch.equal(got.cpu(), expected(q, bounds, bt, lens, bs, top, 1, 1))
