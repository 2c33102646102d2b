"""A bound on the lengths may be any integer: what passes the longest length that a call
takes, and int32, is taken as that length."""
import sys

import pytest
import torch

import test_gpu_paged_attention as A

pytestmark = pytest.mark.gpu


def test_bounds_past_32_bits():
    from starkv_b200.kernels.paged_attention import (empty_bounds, paged_attention_decode, select_pages,
                                                     sparse_paged_decode, update_page_bounds)
    q, k, v, bt, sl = A.make([900, 20, 333], 8, 2, seed=60)
    most, least = sys.maxsize, 960                       # 960: the table's tokens
    assert torch.equal(paged_attention_decode(q, k, v, bt, sl, most, 0.1),
                       paged_attention_decode(q, k, v, bt, sl, least, 0.1))
    a, b = empty_bounds(k), empty_bounds(k)
    update_page_bounds(k, a, bt, sl, most, max_new=most)
    update_page_bounds(k, b, bt, sl, 900, max_new=900)
    assert torch.equal(a, b)
    # the scratch is by the table's tokens then
    assert torch.equal(select_pages(q, a, bt, sl, most, 16, 9), select_pages(q, a, bt, sl, least, 16, 9))
    for x, y in zip(sparse_paged_decode(q, k, v, a, bt, sl, most, 0.1, 9),
                    sparse_paged_decode(q, k, v, a, bt, sl, least, 0.1, 9)):
        assert torch.equal(x, y)
