"""CPU checks of the full-rank paged cache's operators: argument refusals (Python wrappers
and C entry points, before any GPU work), workspace sizes, struct layouts."""
import ctypes as C

import pytest
import torch

BF = torch.bfloat16


def caches(nb=4, bs=16, hkv=2, d=128, dtype=BF):
    return torch.zeros(nb, bs, hkv, d, dtype=dtype), torch.zeros(nb, bs, hkv, d, dtype=dtype)


def attend(q=None, k=None, v=None, bt=None, sl=None, **kw):
    from starkv_b200.kernels.paged_attention import paged_attention_decode
    k0, v0 = caches()
    q = torch.zeros(2, 4, 128, dtype=BF) if q is None else q
    return paged_attention_decode(q, k0 if k is None else k, v0 if v is None else v,
                                  torch.zeros(2, 3, dtype=torch.int32) if bt is None else bt,
                                  torch.ones(2, dtype=torch.int32) if sl is None else sl, 48, 0.1, **kw)


@pytest.mark.parametrize("kw,say", [
    (dict(q=torch.zeros(2, 4, 96, dtype=BF)), "query must be"),
    (dict(q=torch.zeros(2, 5, 128, dtype=BF)), "multiple of 2"),
    (dict(q=torch.zeros(2, 4, 128)), "bf16 or f16"),
    (dict(q=torch.zeros(2, 4, 128, dtype=torch.float16)), "same as the cache"),
    (dict(q=torch.zeros(2, 4, 256, dtype=BF)[..., ::2]), "contiguous"),
    (dict(k=torch.zeros(4, 16, 2, 96, dtype=BF)), "64 or 128"),
    (dict(v=torch.zeros(5, 16, 2, 128, dtype=BF)), "same shape"),
    (dict(bt=torch.zeros(3, 3, dtype=torch.int32)), "block_table must be"),
    (dict(sl=torch.ones(3, dtype=torch.int32)), "seq_lens"),
    (dict(pages=torch.zeros(2, 2, 3)), "pages must be"),
    (dict(pages=torch.zeros(2, 1, 3, dtype=torch.int32)), "pages must be"),
    (dict(out=torch.zeros(2, 4, 128)), "out must be"),
    (dict(), "one CUDA device"),
    (dict(return_partial=True, partial=torch.zeros(8 * 130 - 1)), "at least 1040"),
    (dict(return_partial=True, partial=torch.zeros(8 * 130, dtype=BF)), "f32 buffer"),
])
def test_attention_refusals(kw, say):
    with pytest.raises(ValueError, match=say):
        attend(**kw)


def test_attention_refuses_to_write_over_its_query():
    q = torch.zeros(2, 4, 128, dtype=BF)
    with pytest.raises(ValueError, match="query itself"):
        attend(q=q, out=q)


def test_select_and_bounds_refusals():
    from starkv_b200.kernels.paged_attention import (empty_bounds, select_pages, sparse_paged_decode,
                                                     update_page_bounds)
    k, v = caches()
    b = empty_bounds(k)
    assert b.shape == (4, 2, 2, 128)
    q = torch.zeros(2, 4, 128, dtype=BF)
    bt, sl = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for bad, say in ((dict(top=0), "sinks"), (dict(top=2, sinks=2, recent=1), "sinks"), (dict(top=2, sinks=-1), "sinks"),
                     (dict(top=4), "one CUDA device")):
        with pytest.raises(ValueError, match=say):
            select_pages(q, b, bt, sl, 48, 16, **bad)
        with pytest.raises(ValueError, match=say):
            sparse_paged_decode(q, k, v, b, bt, sl, 48, 0.1, **bad)
    with pytest.raises(ValueError, match="both the same"):
        select_pages(q.half(), b, bt, sl, 48, 16, 4)
    with pytest.raises(ValueError, match="same blocks"):
        sparse_paged_decode(q, k, v, b[:3], bt, sl, 48, 0.1, 4)
    with pytest.raises(ValueError, match="contiguous"):
        select_pages(q, torch.zeros(4, 2, 128, 2, dtype=BF).transpose(2, 3), bt, sl, 48, 16, 4)
    with pytest.raises(ValueError, match="bounds must be"):
        update_page_bounds(k, b[:3], bt, sl, 48)
    with pytest.raises(ValueError, match="new_lens"):
        update_page_bounds(k, b, bt, sl, 48, new_lens=torch.ones(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="one CUDA device"):
        update_page_bounds(k, b, bt, sl, 48)


def test_norm_rope_refusals():
    from starkv_b200.kernels.qk_norm_rope import qk_norm_rope, qk_norm_rope_write
    q, k, v = torch.zeros(3, 4, 128, dtype=BF), torch.zeros(3, 2, 128, dtype=BF), torch.zeros(3, 2, 128, dtype=BF)
    pos, cs = torch.zeros(3, dtype=torch.int64), torch.zeros(10, 128, dtype=BF)
    kc, vc = caches()
    slots = torch.zeros(3, dtype=torch.int64)
    w = torch.ones(128)

    def no(say, f, *a, **kw):
        with pytest.raises(ValueError, match=say):
            f(*a, **kw)
    no("64 or 128", qk_norm_rope, torch.zeros(3, 4, 80, dtype=BF), k, pos, cs)
    no("bf16 or f16", qk_norm_rope, q.float(), k, pos, cs)
    no("k must be", qk_norm_rope, q, k.half(), pos, cs)
    no("positions", qk_norm_rope, q, k, pos.float(), cs)
    no("multiple of 16", qk_norm_rope, q, k, pos, torch.zeros(10, 40, dtype=BF))
    no("at most 128", qk_norm_rope, q, k, pos, torch.zeros(10, 256, dtype=BF))
    no("q_weight", qk_norm_rope, q, k, pos, cs, q_weight=w[:64])
    no("one dtype", qk_norm_rope, q, k, pos, cs, q_weight=w, k_weight=w.half())
    no("need k", qk_norm_rope, q, None, pos, cs, k_weight=w)
    no("q_out", qk_norm_rope, q, k, pos, cs, q_out=q[:2])
    no("k_cache and v_cache", qk_norm_rope_write, q, k, v, pos, cs, kc, vc[:3], slots)
    no("v must be", qk_norm_rope_write, q, k, v[:, :1], pos, cs, kc, vc, slots)
    no("slot_mapping", qk_norm_rope_write, q, k, v, pos, cs, kc, vc, slots[:2])
    no("one CUDA device", qk_norm_rope_write, q, k, v, pos, cs, kc, vc, slots)


def test_workspace_sizes():
    from starkv_b200.kernels.paged_attention import select_workspace_bytes, workspace_bytes
    assert workspace_bytes(32, 8, 128, 1) == 0                    # short units are never split
    big = workspace_bytes(32, 8, 128, 1 << 20)
    assert big == workspace_bytes(32, 8, 128, 5000) > 0           # by the number of CTAs, not by the length
    assert workspace_bytes(32, 5, 128, 5000) == 0                 # no such heads
    for g in range(1, 17):                                        # every slot on a 16-byte boundary
        assert workspace_bytes(g, 1, 128, 5000) % 32 == 0
    assert select_workspace_bytes(2, 8, 1000, 16, 63) == 0        # no more pages than are taken
    assert select_workspace_bytes(2, 8, 1024, 16, 63) >= 2 * 8 * 64 * 8


def test_c_entry_points_refuse_before_any_gpu_work():
    from starkv_b200 import _lib
    L = _lib.lib()
    _lib.check_abi()
    A = 4096   # never dereferenced: every call below is refused first
    names = {"attn": (_lib.PagedAttnArgs, L.starkv_paged_attention), "bounds": (_lib.PageBoundsArgs, L.starkv_page_bounds),
             "select": (_lib.SelectPagesArgs, L.starkv_select_pages), "norm": (_lib.NormRopeArgs, L.starkv_norm_rope)}

    def call(which, ws=(None, 0), **change):
        cls, fn = names[which]
        a = cls()
        for f, t in cls._fields_:
            if f in ("m_out", "l_out", "pages", "status", "new_lens") and not (which == "select" and f == "pages"):
                continue
            if t is C.c_void_p:
                setattr(a, f, A)
            elif f.endswith("_stride") or f == "cs_stride0":
                setattr(a, f, 128 if t is C.c_int64 else (C.c_int64 * t._length_)(*[1024] * t._length_))
        base = dict(dtype=1, n=2, num_heads=8, num_kv_heads=2, head_dim=128, num_blocks=9, block_size=16, max_blocks=4,
                    max_seq_len=1000, top=3, scale=0.1, max_new=1, sinks=1, recent=1, w_dtype=2, pos_dtype=5, cs_dtype=2,
                    slot_dtype=5, rot=128, cs_rows=9, eps=1e-6)
        for f, _ in cls._fields_:
            if f in base:
                setattr(a, f, base[f])
        for f, x in change.items():
            setattr(a, f, x)
        args = ws if which in ("attn", "select") else ()
        return fn(bytes(a), *args, None)

    assert L.starkv_paged_attention(None, None, 0, None) == L.starkv_page_bounds(None, None) == 22
    assert L.starkv_select_pages(None, None, 0, None) == L.starkv_norm_rope(None, None) == 22
    assert L.starkv_sparse_paged_attention(None, None, 0, 0, 1, 1, None, 0, None) == 22
    for which in ("attn", "bounds", "select"):
        assert call(which, n=-1) == call(which, head_dim=96) == call(which, block_size=0) == 22
        assert call(which, max_seq_len=0) == call(which, num_kv_heads=0) == 22
        assert call(which, dtype=2) == call(which, dtype=3) == 101
        assert call(which, block_table=None) == 22
    assert call("norm", head_dim=96) == call("norm", rot=24) == call("norm", rot=144) == call("norm", n=-1) == 22
    assert call("norm", dtype=2) == call("norm", cs_dtype=3) == call("norm", pos_dtype=2) == call("norm", w_dtype=4) == 101
    assert call("norm", slot_dtype=2) == 101
    assert call("norm", v_cache=None) == call("norm", positions=None) == 22
    assert call("norm", query=A + 8) == call("norm", cs_stride0=130) == call("norm", k_weight=A + 4) == 100
    assert call("norm", n=0) == 0
    assert call("attn", num_heads=9) == call("attn", scale=0.0) == call("attn", scale=float("nan")) == 22
    assert call("attn", m_out=A) == 22                                    # l_out is missing
    assert call("attn", query=A + 8) == call("attn", k_stride=(C.c_int64 * 3)(1024, 100, 128)) == 100
    assert call("attn", max_seq_len=1000, max_blocks=100) == 102          # workspace
    assert call("attn", n=0) == call("bounds", n=0) == call("select", n=0) == call("bounds", max_new=0) == 0
    assert call("bounds", max_new=-1) == 22
    assert call("bounds", bounds=A + 2) == 100
    assert call("select", sinks=3) == call("select", top=0) == call("select", recent=-1) == 22
    assert call("select") == 102
    assert call("select", ws=(A + 4, 1 << 20)) == 100


def test_full_layer_and_model_refusals():
    from starkv_b200.full_layer import FullAttentionLayer
    from starkv_b200.model import ModelConfig, StarKVModel
    w = lambda h: torch.zeros(h * 128, 64, dtype=BF)  # noqa: E731
    wo, cs = torch.zeros(64, 6 * 128, dtype=BF), torch.zeros(8, 128, dtype=BF)
    one = torch.ones(128, dtype=BF)
    for kw, say in ((dict(world=2), "split over 2"), (dict(q_norm=one), "both"), (dict(top_pages=1), "at least 2")):
        with pytest.raises(ValueError, match=say):
            FullAttentionLayer(w(6), w(3), w(3), wo, cs, **kw)
    with pytest.raises(ValueError, match="do not group"):
        FullAttentionLayer(w(6), w(4), w(4), wo, cs)
    layer = FullAttentionLayer(w(6), w(3), w(3), wo, cs, top_pages=4)
    assert layer.bytes_per_token() == (2 + 2 / 16) * 3 * 256
    with pytest.raises(ValueError, match="cover"):
        layer.prefill(torch.zeros(3, 64, dtype=BF), None, [2], None, None)
    with pytest.raises(ValueError, match="block_table"):
        layer.prefill(torch.zeros(3, 64, dtype=BF), None, [3], None, None)
    for kw, say in ((dict(full_attention="flash"), "stock"), (dict(full_top_pages=4), "need full_attention"),
                    (dict(full_attention="paged", full_top_pages=4, attn_parallel="context"), "whole sequence")):
        with pytest.raises(ValueError, match=say):
            StarKVModel(ModelConfig(layers=1), "cpu", **kw)
    with pytest.raises(ValueError, match="qk_norm"):
        StarKVModel(ModelConfig(layers=1, qk_norm=True), "cpu")
