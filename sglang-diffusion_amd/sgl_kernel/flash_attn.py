"""`flash_attn_varlen_func` with the reference's signature
(sgl-kernel/python/sgl_kernel/flash_attn.py:228-311), and `flash_attn_with_kvcache` beside it, issuing
`torch.ops.sgl_kernel.fwd` and `fwd_paged_fp8`."""
from __future__ import annotations

import torch

from . import _ops  # noqa: F401

_fwd_paged_fp8 = torch.ops.sgl_kernel.fwd_paged_fp8.default  # (looked up once)


def is_fa3_supported(device=None) -> bool:
    """The MI355X kernel serves the same call; kept for callers that probe it."""
    return torch.cuda.is_available()


def flash_attn_varlen_func(q, k, v, cu_seqlens_q=None, cu_seqlens_k=None, max_seqlen_q=None,
                           max_seqlen_k=None, seqused_q=None, seqused_k=None, page_table=None,
                           softmax_scale=None, causal=False, qv=None, q_descale=None, k_descale=None,
                           v_descale=None, window_size=(-1, -1), attention_chunk=0, softcap=0.0,
                           num_splits=1, pack_gqa=None, sm_margin=0, return_softmax_lse=False,
                           sinks=None, score_mod=None, aux_tensors=None, ver=3):
    if max_seqlen_q is None or max_seqlen_k is None:
        raise ValueError("max_seqlen_q and max_seqlen_k are required for FA3")
    if score_mod is not None or aux_tensors is not None:
        raise NotImplementedError("score_mod / aux_tensors are not implemented")
    if softmax_scale is None:
        softmax_scale = (q.shape[-1] + (qv.shape[-1] if qv is not None else 0)) ** (-0.5)
    attention_chunk = 0 if attention_chunk is None else int(attention_chunk)
    out, softmax_lse, *rest = torch.ops.sgl_kernel.fwd.default(
        q, k, v, None, None, qv, None, cu_seqlens_q, cu_seqlens_k, None, seqused_q, seqused_k,
        max_seqlen_q, max_seqlen_k, page_table, None, None, None, None, None,
        q_descale, k_descale, v_descale, softmax_scale, causal, window_size[0], window_size[1],
        attention_chunk, softcap, is_rotary_interleaved=False, scheduler_metadata=None,
        num_splits=num_splits, pack_gqa=pack_gqa, sm_margin=sm_margin, sinks=sinks)
    return (out, softmax_lse, *rest) if return_softmax_lse else out


def flash_attn_with_kvcache(q, k_cache, v_cache, k=None, v=None, qv=None, rotary_cos=None, rotary_sin=None,
                            cache_seqlens=None, cache_batch_idx=None, cache_leftpad=None, page_table=None,
                            cu_seqlens_q=None, cu_seqlens_k_new=None, max_seqlen_q=None, rotary_seqlens=None,
                            q_descale=None, k_descale=None, v_descale=None, softmax_scale=None, causal=False,
                            window_size=(-1, -1), attention_chunk=None, softcap=0.0, rotary_interleaved=True,
                            scheduler_metadata=None, num_splits=0, pack_gqa=None, sm_margin=0,
                            return_softmax_lse=False, sinks=None, score_mod=None, aux_tensors=None, ver=3):
    """Attention of the newest tokens of each sequence over a paged cache in 8 bits.

    `k_cache`, `v_cache` e4m3 [blocks, block_size, Hk, D] (any strides, D contiguous) with `k_descale`,
    `v_descale` fp32 [blocks, Hk]: one positive scale for each block of tokens and head (the interface's
    own count sequences and heads); value scales outside [2^-64, 2^120] count as the nearer end.
    `page_table` int32 [B, blocks of a sequence], `cache_seqlens` int32 [B] (or one int) counts the new
    tokens too: they are in the cache already (`store_kv_cache_fp8`).  `q` bf16 [B, S, H, D], or packed
    [T, H, D] with `cu_seqlens_q`; rows of a packed q behind the last sequence are not written.  New token
    i of n stands at cache_seqlens - n + i; `causal` hides later keys, `window_size` (w, 0) also those more
    than w back.
    A row that sees no key gives 0, and -inf as its log-sum-exp (fp32 [H, T] or [B, H, S]).  Scores, sums
    and the log-sum-exp are fp32; softmax weights are rounded to half (2^-11) for the product with the
    values, and the output to bf16 (2^-8).
    Everything else of the signature raises RuntimeError instead of being ignored; `num_splits`,
    `pack_gqa` and `sm_margin` are hints that this kernel does not need."""
    if score_mod is not None or aux_tensors is not None:
        raise NotImplementedError("score_mod / aux_tensors are not implemented")
    if page_table is None:
        raise RuntimeError("flash_attn_with_kvcache: only paged caches are implemented (page_table)")
    if k_cache.dtype != torch.float8_e4m3fn:
        raise RuntimeError("flash_attn_with_kvcache: only float8_e4m3fn caches are implemented")
    if not (k is None and v is None and qv is None and rotary_cos is None and rotary_sin is None
            and cache_batch_idx is None and cache_leftpad is None and cu_seqlens_k_new is None
            and rotary_seqlens is None and q_descale is None and sinks is None and attention_chunk in (None, 0)
            and softcap == 0.0):
        raise RuntimeError("flash_attn_with_kvcache: k / v / qv / rotary_* / cache_batch_idx / cache_leftpad / "
                           "cu_seqlens_k_new / q_descale / sinks / attention_chunk / softcap are not implemented for "
                           "an 8-bit cache")
    if isinstance(cache_seqlens, int):
        cache_seqlens = torch.full((page_table.shape[0],), cache_seqlens, dtype=torch.int32, device=q.device)
    out, softmax_lse = _fwd_paged_fp8(
        q, k_cache, v_cache, k_descale, v_descale, page_table, cache_seqlens, cu_seqlens_q, max_seqlen_q, softmax_scale,
        causal, window_size[0], window_size[1])
    if not return_softmax_lse:
        return out
    empty = softmax_lse.new_empty(0)
    return out, softmax_lse, empty, empty
