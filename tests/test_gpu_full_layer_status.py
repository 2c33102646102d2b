"""Device errors of the full-rank layer's kernels reach its user: bad block ids, slots and
positions, in calls and in replayed graphs; a clean step leaves none."""
import pytest
import torch

from test_gpu_full_layer import HID, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top", [None, 4])
@pytest.mark.parametrize("what", ["block", "slot", "position"])
def test_errors_are_recorded(top, what):
    from starkv_b200.full_layer import FullAttentionLayer
    w, norms, cs = weights(8, 2, seed=4)
    dev = cs.device
    layer = FullAttentionLayer(*w, cs, top_pages=top, **norms)
    cache = layer.allocate_cache(21)
    bt = torch.arange(1, 21, dtype=torch.int32, device=dev).view(2, 10)
    hidden = torch.randn(2, HID, device=dev).to(torch.bfloat16)
    sl = torch.tensor([150, 33], dtype=torch.int32, device=dev)
    slots = bt[torch.arange(2, device=dev), (sl.long() - 1) // 16].long() * 16 + (sl.long() - 1) % 16
    pos = sl.long() - 1
    layer.forward(hidden, pos, cache, bt, sl, 160, slots)
    assert layer.read_status() == 0
    bad_bt, bad_pos, bad_slots = bt.clone(), pos.clone(), slots.clone()
    if what == "block":
        bad_bt[1, 0] = 21
    elif what == "slot":
        bad_slots[0] = 21 * 16
    else:
        bad_pos[0] = cs.shape[0]
    layer.forward(hidden, bad_pos, cache, bad_bt, sl, 160, bad_slots)
    assert layer.read_status(reset=False) == 105 and layer.read_status() == 105 and layer.read_status() == 0
    layer.forward(hidden, pos, cache, bt, sl, 160, slots)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        layer.forward(hidden, bad_pos, cache, bad_bt, sl, 160, bad_slots)
    assert layer.read_status() == 0
    g.replay()
    assert layer.read_status() == 105


def test_errors_of_a_prefill_and_of_a_rank():
    from starkv_b200.full_layer import FullAttentionLayer, FullContextLayer
    w, norms, cs = weights(8, 2, seed=5)
    dev = cs.device
    hidden = torch.randn(40, HID, device=dev).to(torch.bfloat16)
    bt = torch.arange(1, 4, dtype=torch.int32, device=dev)[None]
    t = torch.arange(40, device=dev)
    for top, spoil in ((None, "slot"), (4, "block")):
        layer = FullAttentionLayer(*w, cs, top_pages=top, **norms)
        cache = layer.allocate_cache(4)
        layer.prefill(hidden, t, [40], cache, t + 16, block_table=bt)
        assert layer.read_status() == 0
        layer.prefill(hidden, t, [40], cache, t + (64 if spoil == "slot" else 16),
                      block_table=bt + (2 if spoil == "block" else 0))
        assert layer.read_status() == 105
    rank = FullContextLayer(*w, cs, rank=0, world=1, **norms)
    cache = rank.allocate_cache(4)
    sl = torch.tensor([40], dtype=torch.int32, device=dev)
    rank.forward(hidden[:1], t[39:], cache, bt, sl, 48, t[39:] + 16)
    assert rank.read_status() == 0
    rank.forward(hidden[:1], t[39:], cache, bt + 1, sl, 48, t[39:] + 16)
    assert rank.read_status() == 105
