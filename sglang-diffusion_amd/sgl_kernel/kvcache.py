"""What stands around a paged 8-bit key/value cache: block tables and slot maps built on the GPU, and
the store that rounds keys and values into the cache.  `flash_attn_with_kvcache` reads it."""
from __future__ import annotations

from typing import Optional

import torch

from . import _ops  # noqa: F401

# (looked up once)
_kv_block_plan = torch.ops.sgl_kernel.kv_block_plan.default
_store_kv_cache_fp8 = torch.ops.sgl_kernel.store_kv_cache_fp8.default


def kv_block_plan(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                  free_blocks: torch.Tensor, free_begin: torch.Tensor, block_size: int, num_blocks: int,
                  slot_mapping: torch.Tensor, positions: torch.Tensor, cu_seqlens_q: torch.Tensor,
                  seq_lens: torch.Tensor, free_end: torch.Tensor, status: torch.Tensor) -> None:
    """One step's block tables and slot maps from request lengths, without a host round trip.

    Request b holds `context_lens[b]` tokens in the blocks its row of `block_table` names and gets
    `new_lens[b]` more (int32).  The blocks that takes besides come from `free_blocks`, from entry
    `free_begin[0]` on, in the order of the requests, and are written into the table (in place).
    Written: `slot_mapping` and `positions` (int64, one entry for each new token; -1 and 0 behind the
    last), `cu_seqlens_q` [B + 1], `seq_lens` [B], `free_end` [1], and `status` [3] (int32): blocks that
    are lacking, tokens that `slot_mapping` has no room for, requests that outgrow their row.  If any
    of them is not 0, nothing is given to anybody: the table stays, every slot is -1,
    `seq_lens` = `context_lens` and `free_end` = `free_begin`.
    Outputs are other memory than the inputs; copy `seq_lens` and `free_end` back for the next step.
    At most 4096 requests in one call."""
    _kv_block_plan(
        context_lens, new_lens, block_table, free_blocks, free_begin, block_size, num_blocks, slot_mapping,
        positions, cu_seqlens_q, seq_lens, free_end, status)


def store_kv_cache_fp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor,
                       query: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                       inv_freq: Optional[torch.Tensor] = None, attn_factor: float = 1.0,
                       is_neox: bool = True, query_out: Optional[torch.Tensor] = None) -> None:
    """`key`, `value` [T, Hk, D] bf16 into e4m3 caches [blocks, block_size, Hk, D] at `slot_mapping` (int64;
    tokens with a slot outside the pool are skipped), with one power-of-two scale for each block and
    head in `k_scale`, `v_scale` [blocks, Hk] fp32.  A call that writes a block's first token starts
    its scale anew; any other can raise it, and rounds the block's earlier codes to the larger step.
    Tokens may come in any order, with skipped ones between them (those of a block that follow each other
    are fastest); no slot is given twice.  A call keeps what a block holds before the smallest place that
    it writes there, and nothing behind it.

    With `positions` and `inv_freq` the keys are rotated first (as `rotary_embedding_scaled` does,
    rounded to bf16 as it does), and `query` [T, H, D], if given, is rotated in the same launch: into
    `query_out`, or in place.  Caches, scales and `query_out` that overlap each other or the inputs in
    any other way raise."""
    if query is not None and query_out is None:
        query_out = query
    _store_kv_cache_fp8(
        key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping, query, positions, inv_freq, attn_factor,
        is_neox, query_out)
