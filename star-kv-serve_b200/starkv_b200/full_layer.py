"""A full-rank attention layer (one the checkpoint leaves uncompressed) on this library's
kernels:

    q, k, v = hidden . Wqkv^T                     plain library GEMM
    q, k    = rotary(norm(q)), rotary(norm(k))    per-head RMS norms where the model has
    cache  <- k, v at slot_mapping                them; one launch with the write
    attn    = paged decode(q, cache)              all pages, or the best `top_pages` of
                                                  each sequence and KV head
    out     = attn . Wo^T                         plain library GEMM

The reference runs its engine's stock attention in these layers. Query heads may share KV
heads. Tensor parallel over KV heads (split evenly, o_proj partial sums all-reduced), or
with the pages of every sequence split over the ranks (FullContextLayer), as the
compressed layers' StarKVAttentionLayer and StarKVContextLayer.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import context_parallel
from .collectives import all_reduce_
from .kernels import paged_attention as pa
from .kernels.prefill import prefill_attention
from .kernels.qk_norm_rope import qk_norm_rope_write

HEAD_DIM = 128


class FullAttentionLayer:
    """The layer on one rank of a tensor-parallel group of `world` ranks (1: whole).

    wq [Hq * 128, hidden], wk / wv [Hkv * 128, hidden], wo [hidden, Hq * 128]; q_norm /
    k_norm [128]: weights of the per-head norms (both or none). top_pages: decode over
    that many pages per sequence and KV head, chosen by the bounds of their keys (None:
    over all); the first and the last page are always among them."""

    def __init__(self, wq, wk, wv, wo, cos_sin_cache, rank: int = 0, world: int = 1, group=None, q_norm=None,
                 k_norm=None, eps: float = 1e-6, top_pages: int | None = None):
        H, Hkv = wq.shape[0] // HEAD_DIM, wk.shape[0] // HEAD_DIM
        if H % Hkv:
            raise ValueError(f"{H} query heads do not group over {Hkv} KV heads")
        if Hkv % world:
            raise ValueError(f"{Hkv} KV heads do not split over {world} ranks")
        if (q_norm is None) != (k_norm is None):
            raise ValueError("give both q_norm and k_norm or neither")
        if top_pages is not None and top_pages < 2:
            raise ValueError("top_pages must be at least 2 (the first and the last page are always read)")
        hl, kl = H // world, Hkv // world
        q, kv = slice(rank * hl * HEAD_DIM, (rank + 1) * hl * HEAD_DIM), slice(rank * kl * HEAD_DIM, (rank + 1) * kl * HEAD_DIM)
        self.wqkv = torch.cat([wq[q], wk[kv], wv[kv]]).contiguous()
        self.wo = wo[:, q].contiguous()
        self.heads, self.kv_heads, self.world, self.group = hl, kl, world, group
        self.cos_sin_cache = cos_sin_cache
        self.q_norm, self.k_norm, self.eps, self.top_pages = q_norm, k_norm, eps, top_pages
        self.scale = HEAD_DIM ** -0.5
        self.status = torch.zeros(1, dtype=torch.int32, device=self.wqkv.device)

    def read_status(self, reset: bool = True) -> int:
        """The first device error that the layer's kernels recorded since the last reset, 0 if
        none: 105 for a block id, slot or position outside its tensor, 106 for a wait that ran
        out (the selection's lists are -1 then). Synchronises; also after a graph's replay."""
        code = int(self.status)
        if reset and code:
            self.status.zero_()
        return code

    def allocate_cache(self, num_blocks: int, block_size: int = 16) -> tuple:
        """(k_cache, v_cache), and the page bounds behind them with top_pages."""
        k, v = pa.empty_cache(num_blocks, block_size, self.kv_heads, HEAD_DIM, self.wqkv.dtype, self.wqkv.device)
        return (k, v) if self.top_pages is None else (k, v, pa.empty_bounds(k))

    def bytes_per_token(self, block_size: int = 16) -> float:
        """Cache bytes of one token on this rank."""
        rows = 2.0 if self.top_pages is None else 2.0 + 2.0 / block_size
        return rows * self.kv_heads * HEAD_DIM * self.wqkv.element_size()

    def _project(self, hidden, positions, cache, slot_mapping, k_out=None):
        """Rotated queries [n, heads, 128] and values; keys and values go into the cache."""
        n, H, K = hidden.shape[0], self.heads, self.kv_heads
        qkv = F.linear(hidden, self.wqkv).view(n, H + 2 * K, HEAD_DIM)
        q, k, v = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
        q = qk_norm_rope_write(q, k, v, positions, self.cos_sin_cache, cache[0], cache[1], slot_mapping,
                               q_weight=self.q_norm, k_weight=self.k_norm, eps=self.eps, k_out=k_out, status=self.status)
        return q, v

    def _o_proj(self, attn, reduce: bool):
        out = F.linear(attn.reshape(attn.shape[0], -1), self.wo)
        if self.world > 1 and reduce:
            all_reduce_(out, group=self.group)
        return out

    def forward(self, hidden: torch.Tensor, positions: torch.Tensor, cache: tuple, block_table: torch.Tensor,
                seq_lens: torch.Tensor, max_seq_len: int, slot_mapping: torch.Tensor, reduce: bool = True):
        """Decode step of n sequences, one new token each (hidden [n, hidden] at `positions`,
        written at `slot_mapping`; a negative slot and a length of 0 mark a padding row,
        whose attention output is zero); returns the o_proj output [n, hidden],
        all-reduced over the group unless `reduce` is False."""
        q, _ = self._project(hidden, positions, cache, slot_mapping)
        if self.top_pages is None:
            attn = pa.paged_attention_decode(q, cache[0], cache[1], block_table, seq_lens, max_seq_len, self.scale,
                                             status=self.status)
        else:
            pa.update_page_bounds(cache[0], cache[2], block_table, seq_lens, max_seq_len, status=self.status)
            attn, _ = pa.sparse_paged_decode(q, *cache, block_table, seq_lens, max_seq_len, self.scale, self.top_pages,
                                             status=self.status)
        return self._o_proj(attn, reduce)

    def prefill(self, hidden: torch.Tensor, positions: torch.Tensor, prompt_lens: list[int], cache: tuple,
                slot_mapping: torch.Tensor, block_table: torch.Tensor | None = None, reduce: bool = True):
        """Whole prompts with nothing cached before them, back to back in hidden [T,
        hidden]: keys and values written, every prompt attends causally over itself.
        `block_table` (one row per prompt) is needed with top_pages, for the bounds of the
        prompts' pages."""
        T = hidden.shape[0]
        if sum(prompt_lens) != T:
            raise ValueError("prompt_lens must cover the T tokens of hidden")
        if self.top_pages is not None and block_table is None:
            raise ValueError("prefill with top_pages needs the prompts' block_table")
        k = hidden.new_empty((T, self.kv_heads, HEAD_DIM))
        q, v = self._project(hidden, positions, cache, slot_mapping, k_out=k)
        if self.top_pages is not None and T:
            longest = max(prompt_lens)
            lens = torch.tensor(prompt_lens, dtype=torch.int32, device=hidden.device)
            pa.update_page_bounds(cache[0], cache[2], block_table, lens, longest, max_new=longest, status=self.status)
        return self._o_proj(prefill_attention(q, k, v, prompt_lens, self.scale, status=self.status), reduce)


class FullContextLayer(FullAttentionLayer):
    """The decode step with the K/V cache split by pages over `world` ranks: page p of
    every sequence lives on rank p % world (starkv_b200.context_parallel). Every rank
    keeps the whole layer; the ranks' partial attentions are all-gathered and combined
    exactly, and o_proj runs on every rank with no all-reduce. Keys are rotated by their
    global position before they are written, so the cache needs no other table."""

    def __init__(self, wq, wk, wv, wo, cos_sin_cache, rank: int = 0, world: int = 1, group=None, q_norm=None,
                 k_norm=None, eps: float = 1e-6):
        super().__init__(wq, wk, wv, wo, cos_sin_cache, q_norm=q_norm, k_norm=k_norm, eps=eps)
        self.cp_rank, self.cp_world, self.cp_group = rank, world, group

    def bytes_per_token(self, block_size: int = 16) -> float:
        return super().bytes_per_token(block_size) / self.cp_world

    def forward_partial(self, hidden, positions, cache, block_table, seq_lens, max_seq_len, slot_mapping):
        """This rank's part of a decode step: `positions` are global; block_table,
        seq_lens, max_seq_len and slot_mapping (-1 where another rank owns the page)
        describe its local sequences. Returns (out f32 undivided, m, l)."""
        q, _ = self._project(hidden, positions, cache, slot_mapping)
        return pa.paged_attention_decode(q, cache[0], cache[1], block_table, seq_lens, max_seq_len, self.scale,
                                         return_partial=True, status=self.status)

    def forward(self, hidden, positions, cache, block_table, seq_lens, max_seq_len, slot_mapping, reduce: bool = True):
        """Decode step over this rank's pages, the exchange of the partials and o_proj; the
        same on every rank (`reduce` as in FullAttentionLayer; there is no partial sum)."""
        out, m, l = self.forward_partial(hidden, positions, cache, block_table, seq_lens, max_seq_len, slot_mapping)
        if self.cp_world > 1:
            attn = context_parallel.combine(out, m, l, self.cp_group, dtype=self.wo.dtype)
        else:
            attn = context_parallel.combine_local([(out, m, l)], dtype=self.wo.dtype)
        return self._o_proj(attn, reduce)
