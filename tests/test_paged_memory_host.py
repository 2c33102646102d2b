"""CPU checks of the tensors that the full-rank cache's operators write without looking at
their type: a status that cannot hold an aligned int32 and scratch in pieces are refused."""
import pytest
import torch

from test_paged_attention_host import BF, attend, caches


def bad_status():
    return (torch.zeros(0, dtype=torch.int32), torch.zeros(1, dtype=torch.uint8),
            torch.zeros(9, dtype=torch.uint8)[1:])


def calls():
    """Every operator with one keyword argument more."""
    from starkv_b200.kernels import paged_attention as pa
    from starkv_b200.kernels import qk_norm_rope as nr
    k, v = caches()
    b = pa.empty_bounds(k)
    q, pos = torch.zeros(2, 4, 128, dtype=BF), torch.zeros(2, dtype=torch.int64)
    bt, sl = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    cs = torch.zeros(10, 128, dtype=BF)
    return {
        "paged_attention_decode": lambda **kw: attend(**kw),
        "select_pages": lambda **kw: pa.select_pages(q, b, bt, sl, 48, 16, 2, **kw),
        "sparse_paged_decode": lambda **kw: pa.sparse_paged_decode(q, k, v, b, bt, sl, 48, 0.1, 2, **kw),
        "update_page_bounds": lambda **kw: pa.update_page_bounds(k, b, bt, sl, 48, **kw),
        "qk_norm_rope": lambda **kw: nr.qk_norm_rope(q, None, pos, cs, **kw),
        "qk_norm_rope_write": lambda **kw: nr.qk_norm_rope_write(q, q[:, :2], q[:, :2], pos, cs, k, v, pos, **kw),
    }


@pytest.mark.parametrize("name", ["paged_attention_decode", "select_pages", "sparse_paged_decode", "update_page_bounds",
                                  "qk_norm_rope", "qk_norm_rope_write"])
def test_status_must_hold_an_int32(name):
    for t in bad_status():
        with pytest.raises(ValueError, match=f"{name}: status must hold an int32"):
            calls()[name](status=t)
    with pytest.raises(ValueError, match="one CUDA device"):   # the next check: the status was taken
        calls()[name](status=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("name", ["paged_attention_decode", "select_pages", "sparse_paged_decode"])
def test_scratch_must_be_in_one_piece(name):
    with pytest.raises(ValueError, match=f"{name}: ws must be contiguous"):
        calls()[name](ws=torch.zeros(1 << 16, 2, dtype=torch.uint8)[:, 0])
    with pytest.raises(ValueError, match="one CUDA device"):
        calls()[name](ws=torch.zeros(1 << 16, dtype=torch.uint8))
