"""Decode attention over a paged full-rank K/V cache, whole or over selected pages, on
the sm_100a library.

The layers that a STAR-KV checkpoint leaves full-rank keep plain keys and values (the
reference runs its engine's stock attention there). Their cache is a pair of tensors
``[num_blocks, block_size, H_kv, head_dim]`` of any strides with a contiguous last
dimension: tokens before heads, or heads before tokens (``empty_cache``, whose page of a
head is one contiguous run). head_dim 64 or 128, bf16 or f16.

    paged_attention_decode   one new token per sequence, split over the length and joined
    update_page_bounds       per-page smallest / largest key channel values
    select_pages             the pages whose bounds promise the largest scores
    sparse_paged_decode      select_pages, then the attention over those pages alone

There is no fallback: if the native library is missing the calls raise.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from .. import _lib

HEAD_DIMS = (64, 128)


def empty_cache(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int = 128, dtype=torch.bfloat16,
                device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """Zeroed (k_cache, v_cache) ``[num_blocks, block_size, H_kv, head_dim]`` with each
    head's page contiguous."""
    return tuple(torch.zeros(num_blocks, num_kv_heads, block_size, head_dim, dtype=dtype, device=device).transpose(1, 2)
                 for _ in range(2))


def empty_bounds(k_cache: torch.Tensor) -> torch.Tensor:
    """Zeroed page bounds ``[num_blocks, H_kv, 2, head_dim]`` (lo, hi) of a key cache."""
    nb, _, hkv, d = k_cache.shape
    return torch.zeros(nb, hkv, 2, d, dtype=k_cache.dtype, device=k_cache.device)


_CODES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}   # the cache's element types
_LONGEST = 1 << 30   # tokens of a sequence that a call takes; any larger bound means this one


def _tables(what: str, n: int, block_table: torch.Tensor, seq_lens: torch.Tensor):
    """(block_table, seq_lens) as int32, the lengths contiguous."""
    sizes = block_table.shape
    if len(sizes) != 2 or sizes[0] != n or seq_lens.shape != (n,):
        raise ValueError(f"{what}: block_table must be [{n}, max_blocks] and seq_lens [{n}]")
    if block_table.dtype is not torch.int32:
        block_table = block_table.to(torch.int32)
    if seq_lens.dtype is not torch.int32 or not seq_lens.is_contiguous():
        seq_lens = seq_lens.to(torch.int32).contiguous()
    return block_table, seq_lens


def _refuse_memory(what: str, ws: torch.Tensor | None, status: torch.Tensor | None) -> None:
    """The kernels write ws.nbytes in a row, and one aligned int32 of status."""
    if ws is not None and not ws.is_contiguous():
        raise ValueError(f"{what}: ws must be contiguous")
    _lib.refuse_status(what, status)


def _refuse_cache(what: str, name: str, cache: torch.Tensor, dtype: torch.dtype) -> None:
    """The error for a cache tensor that a call does not take, if it does not."""
    if cache.dim() != 4 or cache.shape[3] not in HEAD_DIMS or cache.stride(3) != 1:
        raise ValueError(f"{what}: {name} must be [num_blocks, block_size, H_kv, 64 or 128], last dimension contiguous")
    if cache.dtype is not dtype or dtype not in _CODES:
        raise ValueError(f"{what}: all tensors must be bf16 or f16, the same as the cache")


def _query_sizes(what: str, query: torch.Tensor, num_kv_heads: int, head_dim: int):
    sizes = query.shape
    if len(sizes) != 3 or sizes[2] != head_dim or sizes[1] == 0 or sizes[1] % num_kv_heads or query.stride(2) != 1:
        raise ValueError(f"{what}: query must be [n, multiple of {num_kv_heads}, {head_dim}], last dimension contiguous")
    return sizes


def paged_attention_decode(
    query: torch.Tensor,          # [n, H_q, head_dim], rotation applied
    k_cache: torch.Tensor,        # [num_blocks, block_size, H_kv, head_dim]
    v_cache: torch.Tensor,        # the same shape
    block_table: torch.Tensor,    # [n, max_blocks] int32
    seq_lens: torch.Tensor,       # [n] int32, including the token just written
    max_seq_len: int,             # host-side bound on seq_lens (longer sequences are cut to it)
    scale: float,
    *,
    pages: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    return_partial: bool = False,
    partial: torch.Tensor | None = None,
    ws: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
):
    """``out[b, h] = softmax_t(scale q[b, h] . K[t]) V[t]`` over sequence b's tokens, query
    head h reading KV head h // (H_q / H_kv): [n, H_q, head_dim] in the cache's dtype. A
    sequence of length 0 gives zeros.

    ``pages`` (int32 [n, H_kv, top], as ``select_pages`` returns them): attend to the
    tokens of these pages of the sequence alone. A negative entry holds no token; each
    listed page counts once per listing; of a sequence with fewer than top pages only as
    many entries are read as it has pages.

    ``out`` may not overlap ``query``: a sequence is read by several CTAs.

    ``return_partial``: ``(out, m, l)`` for ``context_parallel.combine`` - out f32
    undivided, m / l f32 [n, H_q] the largest logit and the sum of exp(logit - m) - as
    views of one packed buffer (``partial``, allocated when not given; with head_dim 64,
    which ``combine`` does not take, three tensors).

    ``ws``: contiguous scratch of this call alone (``workspace_bytes``); by default it is
    allocated on the current stream, so that calls that overlap, or captured graphs
    that are replayed at once, do not share it."""
    return _attend("paged_attention_decode", query, k_cache, v_cache, block_table, seq_lens, max_seq_len, scale, pages,
                   out, return_partial, partial, ws, status)


def _attend(what, query, k_cache, v_cache, block_table, seq_lens, max_seq_len, scale, pages, out, return_partial, partial,
            ws, status, select=None):
    """The checks and the call of the attention; ``select`` = (bounds, sinks, recent): the
    pages are selected first, in the same call of the library."""
    # short on purpose: at small batches the host's part of a call takes longer than the GPU's
    dtype, sizes = query.dtype, k_cache.shape
    ks, vs, qs = k_cache.stride(), v_cache.stride(), query.stride()
    if dtype not in _CODES or len(sizes) != 4 or sizes[3] not in HEAD_DIMS or k_cache.dtype is not dtype \
            or v_cache.dtype is not dtype or v_cache.shape != sizes or ks[3] != 1 or vs[3] != 1:
        _refuse_cache(what, "k_cache", k_cache, dtype)
        _refuse_cache(what, "v_cache", v_cache, dtype)
        raise ValueError(f"{what}: k_cache and v_cache must have the same shape")
    nb, bs, hkv, d = sizes
    n, hq, _ = _query_sizes(what, query, hkv, d)
    block_table, seq_lens = _tables(what, n, block_table, seq_lens)
    top, pg = 0, (0, 0)
    if pages is not None:
        if pages.dim() != 3 or pages.shape[:2] != (n, hkv) or pages.dtype is not torch.int32 or pages.shape[2] == 0:
            raise ValueError(f"{what}: pages must be int32 [{n}, {hkv}, top]")
        if pages.stride(-1) != 1:
            raise ValueError(f"{what}: pages needs a contiguous last dimension")
        top, pg = pages.shape[2], pages.stride()[:2]
    m = l = None
    if return_partial:
        if d == 128:
            nh = n * hq
            if partial is None:
                partial = query.new_empty(nh * 130, dtype=torch.float32)
            elif partial.dtype is not torch.float32 or not partial.is_contiguous() or partial.numel() < nh * 130:
                raise ValueError(f"{what}: partial must be a contiguous f32 buffer of at least {nh * 130} values")
            # context_parallel.partial_views, by strides (three slices and views take 8 us)
            at = partial.storage_offset()
            out = partial.as_strided((n, hq, 128), (hq * 128, 128, 1), at)
            m = partial.as_strided((n, hq), (hq, 1), at + nh * 128)
            l = partial.as_strided((n, hq), (hq, 1), at + nh * 129)
        elif partial is not None:
            raise ValueError(f"{what}: the packed partial buffer holds head_dim 128")
        else:
            out = torch.empty((n, hq, d), dtype=torch.float32, device=query.device)
            m, l = torch.empty((2, n, hq), dtype=torch.float32, device=query.device).unbind(0)
    elif out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    elif out.shape != query.shape or out.dtype is not query.dtype or out.stride(-1) != 1:
        raise ValueError(f"{what}: out must be [{n}, {hq}, {d}] in the cache's dtype, last dimension contiguous")
    if out.data_ptr() == query.data_ptr() and n:
        raise ValueError(f"{what}: out may not be the query itself")
    bounds = None if select is None else select[0]
    max_seq_len = min(int(max_seq_len), _LONGEST)
    _refuse_memory(what, ws, status)
    idx = _lib.same_device(what, query, k_cache, v_cache, block_table, seq_lens, pages, out, ws, status, bounds)
    if n == 0:
        return (out, m, l) if return_partial else out
    if ws is None:
        need = workspace_bytes(hq, hkv, d, top * bs if top else max_seq_len)
        if select is not None:
            need += select_workspace_bytes(n, hkv, min(max_seq_len, block_table.shape[1] * bs), bs, top)
        ws = seq_lens.new_empty((need + 3) // 4) if need else None
    P = _lib.addr
    a = _lib.pack_paged_attn(
        query.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2],
        block_table.data_ptr(), *block_table.stride(), seq_lens.data_ptr(), P(pages), *pg, out.data_ptr(),
        *out.stride()[:2], P(m), P(l), P(status), _CODES[dtype], n, hq, hkv, d, nb, bs, block_table.shape[1], max_seq_len, top, float(scale))
    size = 0 if ws is None else ws.nbytes
    if select is None:
        _lib.launch(what, idx, _lib.lib().starkv_paged_attention, a, P(ws), size)
    else:
        _lib.launch(what, idx, _lib.lib().starkv_sparse_paged_attention, a, bounds.data_ptr(), *bounds.stride()[:2],
                    select[1], select[2], P(ws), size)
    return (out, m, l) if return_partial else out


@lru_cache(maxsize=256)   # the calls' sizes repeat
def workspace_bytes(num_heads: int, num_kv_heads: int, head_dim: int, max_tokens: int) -> int:
    """Scratch of one ``paged_attention_decode`` over at most ``max_tokens`` tokens per sequence."""
    return int(_lib.lib().starkv_paged_attention_workspace_bytes(num_heads, num_kv_heads, head_dim,
                                                                  min(int(max_tokens), _LONGEST)))


@lru_cache(maxsize=256)
def select_workspace_bytes(n: int, num_kv_heads: int, max_seq_len: int, block_size: int, top: int) -> int:
    """Scratch of one ``select_pages``; ``sparse_paged_decode`` takes this and ``workspace_bytes``
    of top * block_size tokens."""
    return int(_lib.lib().starkv_select_pages_workspace_bytes(n, num_kv_heads, min(int(max_seq_len), _LONGEST),
                                                              block_size, top))


def update_page_bounds(k_cache: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                       max_seq_len: int, *, max_new: int = 1, new_lens: torch.Tensor | None = None,
                       status: torch.Tensor | None = None) -> None:
    """``bounds[block, h] = (min, max)`` over the page's tokens of every channel of key head
    h, for the pages that hold each sequence's last ``max_new`` tokens (``new_lens``: int32
    [n], per sequence, at most max_new). Call it after those tokens are written: with
    max_new=1 after a decode step, with the longest prompt after a prefill. Other pages'
    bounds stay as they are."""
    what = "update_page_bounds"
    _refuse_cache(what, "k_cache", k_cache, k_cache.dtype)
    nb, bs, hkv, d = k_cache.shape
    if bounds.shape != (nb, hkv, 2, d) or bounds.dtype is not k_cache.dtype or bounds.stride(-1) != 1 \
            or bounds.stride(-2) != d:
        raise ValueError(f"{what}: bounds must be [{nb}, {hkv}, 2, {d}] in the cache's dtype, (lo, hi) contiguous")
    n = block_table.shape[0]
    block_table, seq_lens = _tables(what, n, block_table, seq_lens)
    if new_lens is not None:
        if new_lens.shape != (n,):
            raise ValueError(f"{what}: new_lens must be [{n}]")
        new_lens = new_lens.to(torch.int32).contiguous()
    _refuse_memory(what, None, status)
    idx = _lib.same_device(what, k_cache, bounds, block_table, seq_lens, new_lens, status)
    a = _lib.pack_page_bounds(
        k_cache.data_ptr(), *k_cache.stride()[:3], bounds.data_ptr(), *bounds.stride()[:2], block_table.data_ptr(),
        *block_table.stride(), seq_lens.data_ptr(), _lib.addr(new_lens), _lib.addr(status), _CODES[k_cache.dtype],
        n, hkv, d, nb, bs, block_table.shape[1], min(int(max_seq_len), _LONGEST), min(int(max_new), _LONGEST))
    _lib.launch(what, idx, _lib.lib().starkv_page_bounds, a)


def _check_bounds(what: str, query, bounds, top, sinks, recent):
    if bounds.dim() != 4 or bounds.shape[2] != 2 or bounds.shape[3] not in HEAD_DIMS:
        raise ValueError(f"{what}: bounds must be [num_blocks, H_kv, 2, 64 or 128]")
    nb, hkv, _, d = bounds.shape
    if bounds.dtype is not query.dtype or query.dtype not in _CODES:
        raise ValueError(f"{what}: query and bounds must be bf16 or f16, both the same")
    if bounds.stride(3) != 1 or bounds.stride(2) != d:
        raise ValueError(f"{what}: the (lo, hi) rows of bounds must be contiguous")
    if top < 1 or sinks < 0 or recent < 0 or sinks + recent > top:
        raise ValueError(f"{what}: need top >= 1 and sinks + recent <= top")
    return nb, hkv, d


def select_pages(query: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                 max_seq_len: int, block_size: int, top: int, *, sinks: int = 1, recent: int = 1,
                 out: torch.Tensor | None = None, ws: torch.Tensor | None = None,
                 status: torch.Tensor | None = None) -> torch.Tensor:
    """The ``top`` pages per sequence and KV head with the largest score
    ``sum_d up[d] hi[d] + down[d] lo[d]``, ``up = sum_g max(q[g], 0)`` and ``down = sum_g min(q[g], 0)``
    over the head's query heads g (for finite lo <= hi this is
    ``sum_{g, d} max(q[g, d] lo[d], q[g, d] hi[d])``):
    int32 [n, H_kv, top], ascending, -1 behind them where a sequence has fewer pages.
    The first ``sinks`` and the last ``recent`` pages are always among them (the last
    page is usually not full, and its bounds need not be up to date while recent >= 1).
    Scores in 64 bits; ties go to the lowest page; a NaN score ranks above all others, also
    that of an infinite bound on a side whose ``up`` or ``down`` is 0: a page whose keys
    overflowed that way is taken first."""
    what = "select_pages"
    nb, hkv, d = _check_bounds(what, query, bounds, top, sinks, recent)
    n, hq, _ = _query_sizes(what, query, hkv, d)
    block_table, seq_lens = _tables(what, n, block_table, seq_lens)
    if out is None:
        out = seq_lens.new_empty((n, hkv, top))
    elif out.shape != (n, hkv, top) or out.dtype is not torch.int32 or out.stride(-1) != 1:
        raise ValueError(f"{what}: out must be int32 [{n}, {hkv}, {top}], last dimension contiguous")
    max_seq_len = min(int(max_seq_len), _LONGEST)
    _refuse_memory(what, ws, status)
    idx = _lib.same_device(what, query, bounds, block_table, seq_lens, out, ws, status)
    if n == 0:
        return out
    if ws is None:
        need = select_workspace_bytes(n, hkv, min(max_seq_len, block_table.shape[1] * block_size), block_size, top)
        ws = seq_lens.new_empty((need + 3) // 4) if need else None
    a = _lib.pack_select_pages(
        query.data_ptr(), *query.stride()[:2], bounds.data_ptr(), *bounds.stride()[:2], block_table.data_ptr(),
        *block_table.stride(), seq_lens.data_ptr(), out.data_ptr(), *out.stride()[:2], _lib.addr(status),
        _CODES[query.dtype], n, hq, hkv, d, nb, int(block_size), block_table.shape[1], max_seq_len, int(top),
        int(sinks), int(recent))
    _lib.launch(what, idx, _lib.lib().starkv_select_pages, a, _lib.addr(ws), 0 if ws is None else ws.nbytes)
    return out


def sparse_paged_decode(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, bounds: torch.Tensor,
                        block_table: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int, scale: float, top: int,
                        *, sinks: int = 1, recent: int = 1, out: torch.Tensor | None = None,
                        ws: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """``select_pages``, then ``paged_attention_decode`` over those pages: (out, pages).
    ``bounds`` as ``update_page_bounds`` keeps them. With top >= the pages of a sequence
    this is the attention over all of it."""
    what = "sparse_paged_decode"
    nb, hkv, d = _check_bounds(what, query, bounds, top, sinks, recent)
    if (nb, hkv, d) != (k_cache.shape[0], *k_cache.shape[2:]):
        raise ValueError(f"{what}: bounds and cache must have the same blocks, heads and head_dim")
    pages = block_table.new_empty((query.shape[0], hkv, top), dtype=torch.int32)
    out = _attend(what, query, k_cache, v_cache, block_table, seq_lens, max_seq_len, scale, pages, out, False, None, ws,
                  status, select=(bounds, int(sinks), int(recent)))
    return out, pages
