"""Per-head RMS norms of queries and keys, their rotation and the write of keys and values
into a paged full-rank cache, in one launch of the sm_100a library.

    y = x * rsqrt(mean(x^2) + eps) * weight      (no weight: y = x)
    out = neox rotation of y by the [cos | sin] row of the token's position

Inside all of it is f32 and rounded once. The rotated width is the table's width (a
multiple of 16, at most head_dim); channels behind it are passed through. There is no
fallback: if the native library is missing the calls raise.
"""
from __future__ import annotations

import torch

from .. import _lib
from .paged_attention import _CODES, HEAD_DIMS, _refuse_cache

_Z3 = (0, 0, 0)


_INDEX = {torch.int32: _lib.I32, torch.int64: _lib.I64}
_FLOAT = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}


def _rows(what: str, name: str, t: torch.Tensor, sizes, dtype):
    """The strides of a [n, heads, head_dim] tensor, checked."""
    st = t.stride()
    if t.shape != sizes or t.dtype is not dtype or st[2] != 1:
        raise ValueError(f"{what}: {name} must be {list(sizes)} in the query's dtype, last dimension contiguous")
    return st


def _run(what, q, k, v, positions, cos_sin_cache, k_cache, v_cache, slot_mapping, q_weight, k_weight, eps, q_out, k_out,
         status):
    # short on purpose: at small batches the host's part of a call takes longer than the GPU's
    q_sizes, dtype, qs = q.shape, q.dtype, q.stride()
    if len(q_sizes) != 3 or q_sizes[2] not in HEAD_DIMS or q_sizes[1] == 0 or qs[2] != 1:
        raise ValueError(f"{what}: q must be [n, heads, 64 or 128], last dimension contiguous")
    if dtype not in _CODES:
        raise ValueError(f"{what}: q, k and v must be bf16 or f16")
    n, hq, d = q_sizes
    hkv, ks, vs, os, kos = 0, _Z3, _Z3, _Z3, _Z3
    if k is not None:
        if k.dim() != 3 or k.shape[1] == 0:
            raise ValueError(f"{what}: k must be [n, KV heads, {d}]")
        hkv = k.shape[1]
        k_sizes = (n, hkv, d)
        ks = _rows(what, "k", k, k_sizes, dtype)
    if positions.shape != (n,) or positions.dtype not in _INDEX:
        raise ValueError(f"{what}: positions must be int32 or int64 [{n}]")
    if cos_sin_cache.dim() != 2 or cos_sin_cache.dtype not in _FLOAT:
        raise ValueError(f"{what}: cos_sin_cache must be a bf16, f16 or f32 [positions, rot]")
    rows, rot = cos_sin_cache.shape
    cs = cos_sin_cache.stride()
    if cs[1] != 1 or rot % 16 or not 0 < rot <= d:
        raise ValueError(f"{what}: cos_sin_cache must be [positions, rot], contiguous rows, rot a multiple of 16 and at "
                         f"most {d}")
    w_dtype = None
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            if w.shape != (d,) or w.dtype not in _FLOAT or not w.is_contiguous():
                raise ValueError(f"{what}: {name} must be a contiguous bf16, f16 or f32 [{d}]")
            if w_dtype not in (None, w.dtype):
                raise ValueError(f"{what}: q_weight and k_weight must share one dtype")
            w_dtype = w.dtype
    nb = bs = slot_dtype = 0
    kcs = vcs = _Z3
    if k_cache is not None:
        sizes, kcs, vcs = k_cache.shape, k_cache.stride(), v_cache.stride()
        if len(sizes) != 4 or sizes[2:] != (hkv, d) or v_cache.shape != sizes or k_cache.dtype is not dtype \
                or v_cache.dtype is not dtype or kcs[3] != 1 or vcs[3] != 1:
            _refuse_cache(what, "k_cache", k_cache, dtype)
            _refuse_cache(what, "v_cache", v_cache, dtype)
            raise ValueError(f"{what}: k_cache and v_cache must both be [num_blocks, block_size, {hkv}, {d}]")
        vs = _rows(what, "v", v, k_sizes, dtype)
        if slot_mapping.shape != (n,) or slot_mapping.dtype not in _INDEX:
            raise ValueError(f"{what}: slot_mapping must be int32 or int64 [{n}]")
        nb, bs = sizes[0], sizes[1]
        slot_mapping, slot_dtype = slot_mapping.contiguous(), _INDEX[slot_mapping.dtype]
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os = (hq * d, d)
    else:
        os = _rows(what, "q_out", q_out, q_sizes, dtype)
    if k_out is not None:
        kos = _rows(what, "k_out", k_out, k_sizes, dtype)
    positions = positions.contiguous()
    _lib.refuse_status(what, status)
    idx = _lib.same_device(what, q, k, v, positions, cos_sin_cache, k_cache, v_cache, slot_mapping, q_weight, k_weight,
                           q_out, k_out, status)
    if n == 0:
        return q_out
    P = _lib.addr
    a = _lib.pack_norm_rope(
        q.data_ptr(), qs[0], qs[1], P(k), ks[0], ks[1], P(v), vs[0], vs[1], q_out.data_ptr(), os[0], os[1],
        P(k_out), kos[0], kos[1], P(q_weight), P(k_weight), positions.data_ptr(), cos_sin_cache.data_ptr(), cs[0],
        P(k_cache), kcs[0], kcs[1], kcs[2], P(v_cache), vcs[0], vcs[1], vcs[2], P(slot_mapping), P(status),
        _CODES[dtype], _FLOAT.get(w_dtype, 0), _INDEX[positions.dtype], _FLOAT[cos_sin_cache.dtype], slot_dtype, n, hq,
        hkv, d, rot, rows, nb, bs, float(eps))
    _lib.launch(what, idx, _lib.lib().starkv_norm_rope, a)
    return q_out


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, cos_sin_cache: torch.Tensor, *,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
                 status: torch.Tensor | None = None):
    """(q_out, k_out): normed and rotated q [n, H_q, head_dim] and k [n, H_kv, head_dim]
    (k None: q alone, k_out None). q_out / k_out may be q / k themselves. A position
    outside the table takes the nearest row and is recorded in ``status``."""
    if k is None and (k_out is not None or k_weight is not None):
        raise ValueError("qk_norm_rope: k_out and k_weight need k")
    if k is not None and k_out is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    q_out = _run("qk_norm_rope", q, k, None, positions, cos_sin_cache, None, None, None, q_weight, k_weight, eps, q_out,
                 k_out, status)
    return q_out, k_out


def qk_norm_rope_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                       cos_sin_cache: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       slot_mapping: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                       k_weight: torch.Tensor | None = None, eps: float = 1e-6, q_out: torch.Tensor | None = None,
                       k_out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Normed and rotated q; the normed, rotated k and v go to
    ``cache[slot // block_size, slot % block_size]`` (and k to ``k_out`` where given, as a
    prefill needs it). A negative slot is not written; a slot past the cache is not written
    and recorded in ``status``. Slots are distinct: of two tokens with the same slot either
    may stay. q_out may be q itself."""
    return _run("qk_norm_rope_write", q, k, v, positions, cos_sin_cache, k_cache, v_cache, slot_mapping, q_weight,
                k_weight, eps, q_out, k_out, status)
