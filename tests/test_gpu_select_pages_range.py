"""Page selection at the ends of bf16's range: scores are 64-bit ones also where the products
of queries and bounds are too small or their sums too large for 32 bits."""
import pytest
import torch

from test_gpu_select_pages import cuda, expected

pytestmark = pytest.mark.gpu

# units scored and selected in one kernel, in two, longer than the selection's shared copy, more units than SMs
SIZES = [(200, 2), (900, 2), (9100, 2), (40, 80), (900, 80)]


def select_and_compare(bounds, q, n, P, tops=(2, 30)):
    from starkv_b200.kernels.paged_attention import select_pages
    dev = bounds.device
    bt = torch.arange(1, P + 1, device=dev, dtype=torch.int32).expand(n, P)
    sl = torch.tensor([P, P - 7] * (n // 2), dtype=torch.int32, device=dev)
    for top in tops:
        got = select_pages(q, bounds, bt, sl, P, 1, top)
        assert torch.equal(got.cpu(), expected(q, bounds, bt, sl.tolist(), 1, top, 1, 1)), top


def make(P, n, seed, D=64):
    dev = cuda()
    g = torch.Generator(device=dev).manual_seed(seed)
    b = torch.randn(P + 1, 2, 2, D, generator=g, device=dev, dtype=torch.float64).sort(2).values
    return b, torch.randn(n, 6, D, generator=g, device=dev, dtype=torch.float64)


@pytest.mark.parametrize("P,n", SIZES)
@pytest.mark.parametrize("size", [1e-23, 1e-30])
def test_products_below_the_range_of_32_bits(P, n, size):
    b, q = make(P, n, P)
    select_and_compare((b * size).bfloat16(), (q * size).bfloat16(), n, P)


@pytest.mark.parametrize("P,n", SIZES)
def test_products_next_to_the_smallest_f32(P, n):
    b, q = make(P, n, P + 1)
    select_and_compare((b * 2e-22).bfloat16(), (q * 1e-22).bfloat16(), n, P)


@pytest.mark.parametrize("P,n", SIZES)
def test_sums_above_the_range_of_32_bits(P, n):
    b, q = make(P, n, P + 2)
    select_and_compare((b * 1e20).bfloat16(), (q * 1e20).bfloat16(), n, P)


@pytest.mark.parametrize("P,n", SIZES)
def test_one_page_above_the_range(P, n):
    """Its terms overflow with both signs; its score is the lowest of all, or the highest."""
    b, q = make(P, n, P + 3)
    q[..., 0], q[..., 1] = 1e20, 1e20
    b[:, :, :, 0:2] *= 1e-20
    b[20, :, :, 0], b[20, :, :, 1] = 1e20, -3e20
    b[31, :, :, 0], b[31, :, :, 1] = 3e20, -1e20
    select_and_compare(b.bfloat16(), q.bfloat16(), n, P)
    b[33, 1, 0, 5] = float("nan")                    # and a true NaN beside them
    select_and_compare(b.bfloat16(), q.bfloat16(), n, P, (2, 3, 30))


@pytest.mark.parametrize("P,n", SIZES)
def test_sums_of_queries_above_the_range(P, n):
    b, q = make(P, n, P + 4)
    q[:, :, 3] = 3e38                                # three heads of a group: 9e38
    b[:, :, :, 3] = b[:, :, :, 3] * 1e-38
    select_and_compare(b.bfloat16(), q.bfloat16(), n, P)
    b[:, :, :, 3] = 0
    select_and_compare(b.bfloat16(), q.bfloat16(), n, P)
