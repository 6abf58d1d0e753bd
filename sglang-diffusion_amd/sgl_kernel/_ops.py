"""`torch.ops.sgl_kernel.*` for MI355X: the reference's op registry, backed by libmi355dit.so.

The reference registers these ops from C++ (`TORCH_LIBRARY_FRAGMENT(sgl_kernel, m)`,
sgl-kernel/csrc/common_extension.cc:21,66-97,134-158 and flash_extension.cc:21-66) and its
Python layers call them as `torch.ops.sgl_kernel.<name>.default(...)`.  Here the same schemas
are defined from Python and each one is implemented for the `CUDA` dispatch key (= HIP devices
under PyTorch-ROCm) by a call through the C ABI of include/mi355_dit.h.  There is no CPU
implementation: CPU tensors hit the dispatcher's "no kernel for backend CPU" error, and a
missing shared object raises on first use.  `torch.library.register_fake` shims give the
shape/dtype rules for tracing, as the reference does in
python/sglang/srt/layers/quantization/fp8_utils.py:69-81 and fp8_kernel.py:2057-2076.

Conventions kept from the reference: `Tensor!` outputs are caller-allocated and written in
place; functional ops allocate their result on the input's device; kernels are enqueued on the
current stream and never synchronise; unsupported arguments raise RuntimeError instead of being
ignored.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from sglang_diffusion_amd import _C

FP8 = torch.float8_e4m3fn

SCHEMAS = {
    # sgl-kernel/csrc/common_extension.cc:134-158 (gemm section)
    "fp8_scaled_mm": "(Tensor mat_a, Tensor mat_b, Tensor scales_a, Tensor scales_b, "
                     "ScalarType out_dtype, Tensor? bias) -> Tensor",
    "fp8_blockwise_scaled_mm": "(Tensor mat_a, Tensor mat_b, Tensor scales_a, Tensor scales_b, "
                               "ScalarType out_dtype) -> Tensor",
    "sgl_per_token_quant_fp8": "(Tensor input, Tensor! output_q, Tensor! output_s) -> ()",
    "sgl_per_token_group_quant_8bit": "(Tensor input, Tensor! output_q, Tensor! output_s, "
                                      "int group_size, float eps, float fp8_min, float fp8_max, "
                                      "bool scale_ue8m0) -> ()",
    "sgl_per_tensor_quant_fp8": "(Tensor input, Tensor! output_q, Tensor! output_s, "
                                "bool is_static) -> ()",
    # sgl-kernel/csrc/common_extension.cc:66-97 (elementwise section)
    "rmsnorm": "(Tensor! output, Tensor input, Tensor weight, float eps, bool enable_pdl) -> ()",
    "fused_add_rmsnorm": "(Tensor! input, Tensor! residual, Tensor weight, float eps, "
                         "bool enable_pdl) -> ()",
    "rotary_embedding": "(Tensor positions, Tensor! query, Tensor!? key, int head_size, "
                        "Tensor cos_sin_cache, bool is_neox) -> ()",
    "apply_rope_pos_ids_cos_sin_cache": "(Tensor q, Tensor k, Tensor! q_rope, Tensor! k_rope, "
                                        "Tensor cos_sin_cache, Tensor pos_ids, bool interleave, "
                                        "bool enable_pdl, Tensor? v, Tensor!? k_buffer, "
                                        "Tensor!? v_buffer, Tensor? kv_cache_loc) -> ()",
    # sgl-kernel/csrc/common_extension.cc:55-56
    "merge_state_v2": "(Tensor v_a, Tensor s_a, Tensor v_b, Tensor s_b, Tensor! v_merged, "
                      "Tensor! s_merged) -> ()",
    # sgl-kernel/csrc/flash_extension.cc:25-63
    "fwd": "(Tensor q, Tensor k, Tensor v, Tensor? k_new, Tensor? v_new, Tensor? q_v, "
           "Tensor? out, Tensor? cu_seqlens_q, Tensor? cu_seqlens_k, Tensor? cu_seqlens_k_new, "
           "Tensor? seqused_q, Tensor? seqused_k, int? max_seqlen_q, int? max_seqlen_k, "
           "Tensor? page_table, Tensor? kv_batch_idx, Tensor? leftpad_k, Tensor? rotary_cos, "
           "Tensor? rotary_sin, Tensor? seqlens_rotary, Tensor? q_descale, Tensor? k_descale, "
           "Tensor? v_descale, float? softmax_scale, bool is_causal, int window_left, "
           "int window_right, int attention_chunk, float softcap, bool is_rotary_interleaved, "
           "Tensor? scheduler_metadata, int num_splits, bool? pack_gqa, int sm_margin, "
           "Tensor? sinks) -> (Tensor, Tensor, Tensor, Tensor)",
    # the paged 8-bit cache that `fwd` reads through page_table: ops of this package, in the
    # conventions of the ones above
    "fwd_paged_fp8": "(Tensor q, Tensor k_cache, Tensor v_cache, Tensor? k_descale, Tensor? v_descale, "
                     "Tensor page_table, Tensor? cache_seqlens, Tensor? cu_seqlens_q, int? max_seqlen_q, "
                     "float? softmax_scale, bool causal, int window_left, int window_right) -> (Tensor, Tensor)",
    "kv_block_plan": "(Tensor context_lens, Tensor new_lens, Tensor! block_table, Tensor free_blocks, "
                     "Tensor free_begin, int block_size, int num_blocks, Tensor! slot_mapping, "
                     "Tensor! positions, Tensor! cu_seqlens_q, Tensor! seq_lens, Tensor! free_end, "
                     "Tensor! status) -> ()",
    "rotary_embedding_scaled": "(Tensor positions, Tensor query, Tensor? key, Tensor inv_freq, "
                               "float attn_factor, bool is_neox, Tensor! query_out, "
                               "Tensor!? key_out) -> ()",
    "store_kv_cache_fp8": "(Tensor key, Tensor value, Tensor! k_cache, Tensor! v_cache, "
                          "Tensor! k_scale, Tensor! v_scale, Tensor slot_mapping, Tensor? query, "
                          "Tensor? positions, Tensor? inv_freq, float attn_factor, bool is_neox, "
                          "Tensor!? query_out) -> ()",
}

_lib = torch.library.Library("sgl_kernel", "FRAGMENT")
for _name, _schema in SCHEMAS.items():
    _lib.define(_name + _schema)


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


# ------------------------------------------------------------------------------------ GEMM --
def _check_mm(mat_a, mat_b, out_dtype, what):
    """Layout preconditions of sgl-kernel/csrc/gemm/fp8_gemm_kernel.cu:1457-1487."""
    _require(mat_a.dim() == 2 and mat_b.dim() == 2, f"{what}: mat_a and mat_b must be 2-D")
    _require(mat_a.dtype == FP8 and mat_b.dtype == FP8, f"{what}: operands must be float8_e4m3fn")
    _require(mat_a.stride(1) == 1, f"{what}: mat_a must be row major")
    _require(mat_b.stride(0) == 1, f"{what}: mat_b must be column major (a [N,K] weight, transposed)")
    _require(mat_a.shape[1] == mat_b.shape[0], f"{what}: inner dimensions differ")
    _require(out_dtype in (torch.bfloat16, torch.float16),
             f"{what}: out_dtype must be bfloat16 or float16")
    _require(mat_a.shape[1] % 16 == 0, f"{what}: K must be a multiple of 16")
    _require(mat_b.shape[1] % 8 == 0, f"{what}: N must be a multiple of 8")


def _fp8_scaled_mm(mat_a, mat_b, scales_a, scales_b, out_dtype, bias):
    _check_mm(mat_a, mat_b, out_dtype, "fp8_scaled_mm")
    M, K = mat_a.shape
    N = mat_b.shape[1]
    _require(scales_a.numel() == M and scales_b.numel() == N,
             "fp8_scaled_mm: scales_a must have M and scales_b N elements")
    _require(scales_a.dtype == torch.float32 and scales_b.dtype == torch.float32,
             "fp8_scaled_mm: scales must be float32")
    _require(scales_a.is_contiguous() and scales_b.is_contiguous(),
             "fp8_scaled_mm: scales must be contiguous")
    if bias is not None:
        _require(bias.numel() == N and bias.dtype == out_dtype and bias.is_contiguous(),
                 "fp8_scaled_mm: bias must be a contiguous [N] tensor of out_dtype")
    out = torch.empty((M, N), dtype=out_dtype, device=mat_a.device)
    if M:
        _C.fp8_scaled_mm(mat_a, mat_b.t(), scales_a, scales_b, bias, out)
    return out


def _fp8_blockwise_scaled_mm(mat_a, mat_b, scales_a, scales_b, out_dtype):
    """scales_a [M, K/128] (either stride order), scales_b [K/128, N/128] (either order):
    sgl-kernel/csrc/gemm/fp8_blockwise_gemm_kernel.cu:374-406."""
    _check_mm(mat_a, mat_b, out_dtype, "fp8_blockwise_scaled_mm")
    M, K = mat_a.shape
    N = mat_b.shape[1]
    kb, nb = (K + 127) // 128, (N + 127) // 128
    _require(tuple(scales_a.shape) == (M, kb), "fp8_blockwise_scaled_mm: scales_a must be [M, ceil(K/128)]")
    _require(tuple(scales_b.shape) == (kb, nb),
             "fp8_blockwise_scaled_mm: scales_b must be [ceil(K/128), ceil(N/128)]")
    _require(scales_a.dtype == torch.float32 and scales_b.dtype == torch.float32,
             "fp8_blockwise_scaled_mm: scales must be float32")
    out = torch.empty((M, N), dtype=out_dtype, device=mat_a.device)
    if M:
        _C.fp8_blockwise_scaled_mm(mat_a, mat_b.t(), scales_a, scales_b, out,
                                   (scales_a.stride(0), scales_a.stride(1)),
                                   (scales_b.stride(0), scales_b.stride(1)))
    return out


# ----------------------------------------------------------------------------------- quant --
def _as_rows(x: torch.Tensor, what: str) -> torch.Tensor:
    _require(x.stride(-1) == 1, f"{what}: last dimension must be contiguous")
    if x.dim() == 2:
        return x
    _require(x.is_contiguous(), f"{what}: inputs with more than 2 dimensions must be contiguous")
    return x.view(-1, x.shape[-1])


def _sgl_per_token_quant_fp8(input, output_q, output_s):
    x = _as_rows(input, "sgl_per_token_quant_fp8")
    _require(input.dtype == torch.bfloat16, "sgl_per_token_quant_fp8: input must be bfloat16")
    _require(output_q.dtype == FP8 and output_q.is_contiguous(),
             "sgl_per_token_quant_fp8: output_q must be contiguous float8_e4m3fn")
    _require(output_s.dtype == torch.float32 and output_s.numel() == x.shape[0],
             "sgl_per_token_quant_fp8: output_s must hold one float32 per token")
    _C.per_token_quant_fp8(x, output_q.view(x.shape), output_s)


def _sgl_per_token_group_quant_8bit(input, output_q, output_s, group_size, eps, fp8_min, fp8_max,
                                    scale_ue8m0):
    x = _as_rows(input, "sgl_per_token_group_quant_8bit")
    _require(input.dtype == torch.bfloat16, "sgl_per_token_group_quant_8bit: input must be bfloat16")
    _require(output_q.dtype == FP8, "sgl_per_token_group_quant_8bit: only float8_e4m3fn output "
                                    "is implemented (int8 is not on the diffusion path)")
    _require(output_q.is_contiguous(), "sgl_per_token_group_quant_8bit: output_q must be contiguous")
    M, K = x.shape
    _require(K % group_size == 0, "sgl_per_token_group_quant_8bit: K must divide by group_size")
    s = output_s if output_s.dim() == 2 else output_s.view(M, K // group_size)
    _require(tuple(s.shape) == (M, K // group_size),
             "sgl_per_token_group_quant_8bit: output_s must be [M, K/group_size]")
    _C.per_token_group_quant_fp8(x, output_q.view(M, K), s, group_size, eps, fp8_min, fp8_max,
                                 scale_ue8m0)


def _sgl_per_tensor_quant_fp8(input, output_q, output_s, is_static):
    _require(input.is_contiguous() and output_q.is_contiguous(),
             "sgl_per_tensor_quant_fp8: tensors must be contiguous")
    _require(input.dtype == torch.bfloat16 and output_q.dtype == FP8,
             "sgl_per_tensor_quant_fp8: bfloat16 -> float8_e4m3fn only")
    _require(output_s.dtype == torch.float32 and output_s.numel() == 1,
             "sgl_per_tensor_quant_fp8: output_s must be one float32")
    _C.per_tensor_quant_fp8(input, output_q, output_s, is_static)


# ------------------------------------------------------------------------------ norm / rope --
def _rmsnorm(output, input, weight, eps, enable_pdl):
    x = _as_rows(input, "rmsnorm")
    o = _as_rows(output, "rmsnorm")
    _require(input.dtype == torch.bfloat16 and output.dtype == torch.bfloat16,
             "rmsnorm: bfloat16 activations only")
    _require(weight.numel() == x.shape[1] and weight.is_contiguous(), "rmsnorm: weight must be [hidden]")
    _C.rmsnorm(o, x, weight, eps)


def _fused_add_rmsnorm(input, residual, weight, eps, enable_pdl):
    _require(input.is_contiguous() and residual.is_contiguous(),
             "fused_add_rmsnorm: input and residual must be contiguous")
    _require(input.dtype == torch.bfloat16 and residual.dtype == torch.bfloat16,
             "fused_add_rmsnorm: bfloat16 only")
    _C.fused_add_rmsnorm(input.view(-1, input.shape[-1]), residual.view(-1, input.shape[-1]),
                         weight, eps)


def _rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox):
    _require(positions.dtype == torch.int64 and positions.is_contiguous(),
             "rotary_embedding: positions must be contiguous int64")
    _require(query.dtype == torch.bfloat16, "rotary_embedding: bfloat16 only")
    _require(cos_sin_cache.dtype in (torch.float32, torch.bfloat16) and cos_sin_cache.is_contiguous(),
             "rotary_embedding: cos_sin_cache must be contiguous float32 or bfloat16")
    _C.rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox)


def _apply_rope_pos_ids_cos_sin_cache(q, k, q_rope, k_rope, cos_sin_cache, pos_ids, interleave,
                                      enable_pdl, v, k_buffer, v_buffer, kv_cache_loc):
    _require(v is None and k_buffer is None and v_buffer is None and kv_cache_loc is None,
             "apply_rope_pos_ids_cos_sin_cache: the fused KV-cache write is an LLM-serving "
             "feature and is not implemented on the diffusion path")
    _require(q.dim() == 3 and k.dim() == 3, "apply_rope_pos_ids_cos_sin_cache: q, k must be [nnz, H, d]")
    _require(cos_sin_cache.dtype == torch.float32, "cos_sin_cache should be float32")
    if q_rope.data_ptr() != q.data_ptr():
        q_rope.copy_(q)
    if k_rope.data_ptr() != k.data_ptr():
        k_rope.copy_(k)
    _require(q_rope.stride(-1) == 1 and q_rope.stride(1) == q_rope.shape[2]
             and k_rope.stride(-1) == 1 and k_rope.stride(1) == k_rope.shape[2],
             "apply_rope_pos_ids_cos_sin_cache: heads must be packed within a token")
    nnz, _, d = q_rope.shape
    qv = q_rope.as_strided((nnz, q_rope.shape[1] * d), (q_rope.stride(0), 1))
    kv = k_rope.as_strided((nnz, k_rope.shape[1] * d), (k_rope.stride(0), 1))
    _C.rotary_embedding(pos_ids.contiguous(), qv, kv, d, cos_sin_cache, not interleave)


# -------------------------------------------------------------------------------- attention --
def _fwd(q, k, v, k_new, v_new, q_v, out, cu_seqlens_q, cu_seqlens_k, cu_seqlens_k_new, seqused_q,
         seqused_k, max_seqlen_q, max_seqlen_k, page_table, kv_batch_idx, leftpad_k, rotary_cos,
         rotary_sin, seqlens_rotary, q_descale, k_descale, v_descale, softmax_scale, is_causal,
         window_left, window_right, attention_chunk, softcap, is_rotary_interleaved,
         scheduler_metadata, num_splits, pack_gqa, sm_margin, sinks):
    """With page_table and e4m3 caches: attention over a paged 8-bit cache (fwd_paged_fp8).  Otherwise
    dense non-causal attention, the only form the diffusion path issues
    (python/sglang/multimodal_gen/runtime/layers/attention/backends/flash_attn.py:517-563).
    Batched [B,S,H,d] inputs, or packed [T,H,d] inputs whose sequences all have the maximum
    length.  Everything the LLM-serving callers use besides that is rejected."""
    if page_table is not None and k.dtype == FP8:
        other = dict(k_new=k_new, v_new=v_new, q_v=q_v, cu_seqlens_k=cu_seqlens_k,
                     cu_seqlens_k_new=cu_seqlens_k_new, seqused_q=seqused_q, kv_batch_idx=kv_batch_idx,
                     leftpad_k=leftpad_k, rotary_cos=rotary_cos, rotary_sin=rotary_sin,
                     seqlens_rotary=seqlens_rotary, q_descale=q_descale, sinks=sinks)
        if any(t is not None for t in other.values()):
            _fail("fwd: arguments not supported with a paged 8-bit cache: "
                  f"{[n for n, t in other.items() if t is not None]}")
        _require(attention_chunk == 0 and softcap == 0.0, "fwd: attention_chunk / softcap are not implemented")
        out, lse = _fwd_paged_fp8(q, k, v, k_descale, v_descale, page_table, seqused_k, cu_seqlens_q, max_seqlen_q,
                                  softmax_scale, is_causal, window_left, window_right, out)
        empty = lse.new_empty(0)
        return out, lse, empty, empty
    unsupported = dict(k_new=k_new, v_new=v_new, q_v=q_v, cu_seqlens_k_new=cu_seqlens_k_new,
                       seqused_q=seqused_q, seqused_k=seqused_k, page_table=page_table,
                       kv_batch_idx=kv_batch_idx, leftpad_k=leftpad_k, rotary_cos=rotary_cos,
                       rotary_sin=rotary_sin, seqlens_rotary=seqlens_rotary, q_descale=q_descale,
                       k_descale=k_descale, v_descale=v_descale, sinks=sinks)
    bad = [n for n, t in unsupported.items() if t is not None]
    _require(not bad, f"fwd: arguments not supported on the diffusion path: {bad}")
    _require(not is_causal, "fwd: causal attention is not implemented (diffusion attention is dense)")
    _require(window_left < 0 and window_right < 0, "fwd: sliding windows are not implemented")
    _require(attention_chunk == 0 and softcap == 0.0, "fwd: attention_chunk / softcap are not implemented")
    _require(q.dtype == torch.bfloat16 and k.dtype == q.dtype and v.dtype == q.dtype,
             "fwd: bfloat16 q, k, v only")
    _require(q.stride(-1) == 1 and k.stride(-1) == 1 and v.stride(-1) == 1,
             "fwd: last dimension of q, k, v must be contiguous")
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    packed = q.dim() == 3
    if packed:
        _require(cu_seqlens_q is not None and cu_seqlens_k is not None and max_seqlen_q and max_seqlen_k,
                 "fwd: packed inputs need cu_seqlens_q/k and max_seqlen_q/k")
        nb = cu_seqlens_q.numel() - 1
        _require(cu_seqlens_k.numel() - 1 == nb, "fwd: cu_seqlens_q and cu_seqlens_k disagree")
        # equal totals <=> every sequence has the maximum length: no device read needed
        _require(q.shape[0] == nb * max_seqlen_q and k.shape[0] == nb * max_seqlen_k,
                 "fwd: ragged packed batches are not implemented; all sequences must have max_seqlen")
        T, H, d = q.shape
        q4 = q.as_strided((nb, max_seqlen_q, H, d), (max_seqlen_q * q.stride(0), q.stride(0), q.stride(1), 1))
        k4 = k.as_strided((nb, max_seqlen_k, k.shape[1], d),
                          (max_seqlen_k * k.stride(0), k.stride(0), k.stride(1), 1))
        v4 = v.as_strided((nb, max_seqlen_k, v.shape[1], d),
                          (max_seqlen_k * v.stride(0), v.stride(0), v.stride(1), 1))
    else:
        _require(q.dim() == 4, "fwd: q must be [B,S,H,d] or [T,H,d]")
        _require(cu_seqlens_q is None and cu_seqlens_k is None,
                 "fwd: cu_seqlens with batched 4-D inputs are not supported")
        q4, k4, v4 = q, k, v
    B, Sq, H, d = q4.shape
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _require(out.shape == q.shape and out.dtype == q.dtype and out.stride(-1) == 1,
                 "fwd: out must match q")
    o4 = out if not packed else out.as_strided(
        (B, Sq, H, d), (Sq * out.stride(0), out.stride(0), out.stride(1), 1))
    lse = torch.empty((B, H, Sq), dtype=torch.float32, device=q.device)
    if B and Sq:
        _C.attention(q4, k4, v4, o4, lse, softmax_scale)
    if packed:  # FA3's packed layout of the log-sum-exp is [H, T]
        lse = lse.permute(1, 0, 2).reshape(H, B * Sq)
    empty = torch.empty(0, dtype=torch.float32, device=q.device)
    return out, lse, empty, empty


# The checks of the operators around the paged cache run at every step of a serving loop, whose
# kernels take a few microseconds: messages are only formed when something is wrong.
def _fail(msg):
    raise RuntimeError(msg)


_ONE = (1,)


def _dense(t, dtype, shape, device):
    return t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.get_device() == device


def _check_cache(what, cache, scale, name, like):
    if not (cache.dtype == FP8 and cache.dim() == 4 and cache.stride(3) == 1):
        _fail(f"{what}: {name}_cache must be [blocks, block_size, heads, head_size] float8_e4m3fn with a "
              "contiguous last dimension")
    if not (scale is not None and scale.dtype == torch.float32 and scale.is_contiguous()
            and scale.shape == (cache.shape[0], cache.shape[2])):
        _fail(f"{what}: the scales of {name}_cache must be contiguous float32 [blocks, heads]")
    if not cache.get_device() == scale.get_device() == like.get_device():
        _fail(f"{what}: all tensors must be on {like.device}")


def _check_ints(what, like, dtype, **tensors):
    device = like.get_device()
    for name, t in tensors.items():
        if not (t.dtype == dtype and t.dim() == 1 and t.is_contiguous()):
            _fail(f"{what}: {name} must be a contiguous 1-D {str(dtype)[6:]} tensor")
        if t.get_device() != device:
            _fail(f"{what}: all tensors must be on {like.device}")


def _check_table(what, table, rows, name, like):
    if not (table.dtype == torch.int32 and table.dim() == 2 and table.shape[0] == rows
            and (table.shape[1] <= 1 or table.stride(1) == 1) and table.get_device() == like.get_device()):
        _fail(f"{what}: {name} must be int32 [sequences, blocks] with contiguous rows, on {like.device}")


def _check_heads(what, x, tokens, name, like):
    if not (x.dtype == torch.bfloat16 and x.dim() == 3 and x.stride(2) == 1 and x.shape[0] == tokens):
        _fail(f"{what}: {name} must be bfloat16 [tokens, heads, head_size] with a contiguous last dimension")
    if x is not like and x.get_device() != like.get_device():
        _fail(f"{what}: all tensors must be on {like.device}")


def _check_inv_freq(what, inv_freq, like):
    if not (inv_freq.dtype in (torch.float64, torch.float32) and inv_freq.dim() == 1 and inv_freq.is_contiguous()
            and inv_freq.get_device() == like.get_device()):
        _fail(f"{what}: inv_freq must be a contiguous 1-D float64 or float32 tensor on {like.device}")


def _check_fwd_paged(q, k_cache, v_cache, k_descale, v_descale, page_table, cache_seqlens, cu_seqlens_q, is_causal,
                     window_left, window_right):
    packed = q.dim() == 3
    if not (q.dtype == torch.bfloat16 and (packed or q.dim() == 4) and q.stride(-1) == 1):
        _fail("fwd: q must be bfloat16 [T,H,d] or [B,S,H,d] with a contiguous last dimension")
    _check_cache("fwd", k_cache, k_descale, "k", q)
    _check_cache("fwd", v_cache, v_descale, "v", q)
    if not (v_cache.shape == k_cache.shape and k_cache.shape[3] == q.shape[-1]):
        _fail("fwd: k_cache and v_cache must have one shape, with the head size of q")
    if cache_seqlens is None:
        _fail("fwd: a paged cache needs the sequences' lengths (cache_seqlens)")
    B = cache_seqlens.numel()
    _check_table("fwd", page_table, B, "page_table", q)
    if packed:
        if cu_seqlens_q is None:
            _fail("fwd: packed q needs cu_seqlens_q")
        _check_ints("fwd", q, torch.int32, cache_seqlens=cache_seqlens, cu_seqlens_q=cu_seqlens_q)
        if cu_seqlens_q.numel() != B + 1:
            _fail("fwd: cu_seqlens_q and cache_seqlens disagree")
    else:
        _check_ints("fwd", q, torch.int32, cache_seqlens=cache_seqlens)
        if cu_seqlens_q is not None or q.shape[0] != B:
            _fail("fwd: batched q needs one sequence for each length and no cu_seqlens_q")
    H, Hk = q.shape[-2], k_cache.shape[2]
    if not (Hk > 0 and H > 0 and H % Hk == 0):
        _fail("fwd: the heads of q must be a multiple of the cache's")
    if not (window_left < 0 and window_right < 0 or is_causal and window_right in (-1, 0)):
        _fail("fwd: sliding windows need causal attention, and end at the token itself")


def _fwd_paged_fp8(q, k_cache, v_cache, k_descale, v_descale, page_table, cache_seqlens, cu_seqlens_q, max_seqlen_q,
                   softmax_scale, is_causal, window_left, window_right, out=None):
    shape, cache, dev = q.shape, k_cache.shape, q.get_device()
    packed = len(shape) == 3
    # the usual call in few steps; whatever is not that is looked at one by one
    scales = cache[0::2]
    if not (q.dtype is torch.bfloat16 and k_cache.dtype is FP8 and v_cache.dtype is FP8 and packed and len(cache) == 4
            and v_cache.shape == cache and cache[3] == shape[2] and shape[1] % max(cache[2], 1) == 0 and shape[1] > 0
            and q.stride(2) == 1 and k_cache.stride(3) == 1 and v_cache.stride(3) == 1
            and (window_left < 0 and window_right < 0 or is_causal and -1 <= window_right <= 0)
            and k_descale is not None and v_descale is not None and cu_seqlens_q is not None
            and cache_seqlens is not None
            and _dense(k_descale, torch.float32, scales, dev) and _dense(v_descale, torch.float32, scales, dev)
            and page_table.dtype is torch.int32 and page_table.stride()[1:] == _ONE
            and _dense(cache_seqlens, torch.int32, page_table.shape[:1], dev)
            and _dense(cu_seqlens_q, torch.int32, (page_table.shape[0] + 1,), dev)
            and k_cache.get_device() == v_cache.get_device() == page_table.get_device() == dev):
        _check_fwd_paged(q, k_cache, v_cache, k_descale, v_descale, page_table, cache_seqlens, cu_seqlens_q, is_causal,
                         window_left, window_right)
    B = page_table.shape[0]
    device = q.device
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif not (out.shape == shape and out.dtype == q.dtype and out.stride(-1) == 1 and out.device == device):
        _fail("fwd: out must match q")
    if packed:
        lse = torch.empty(shape[1], shape[0], dtype=torch.float32, device=device)
        if max_seqlen_q is None:
            max_seqlen_q = shape[0]
    else:
        lse = torch.empty(B, shape[2], shape[1], dtype=torch.float32, device=device)
        max_seqlen_q = shape[1]
    if softmax_scale is None:
        softmax_scale = shape[-1] ** -0.5
    if q.numel() and B:
        _C.paged_attention_fp8(q, k_cache, v_cache, k_descale, v_descale, page_table, cache_seqlens, cu_seqlens_q,
                               max_seqlen_q, out, lse, softmax_scale, is_causal, window_left)
    return out, lse


# --------------------------------------------------------------------- paged 8-bit KV cache --
def _kv_block_plan(context_lens, new_lens, block_table, free_blocks, free_begin, block_size, num_blocks,
                   slot_mapping, positions, cu_seqlens_q, seq_lens, free_end, status):
    what = "kv_block_plan"
    _check_ints(what, slot_mapping, torch.int32, context_lens=context_lens, new_lens=new_lens,
                free_blocks=free_blocks, free_begin=free_begin, cu_seqlens_q=cu_seqlens_q, seq_lens=seq_lens,
                free_end=free_end, status=status)
    _check_ints(what, slot_mapping, torch.int64, slot_mapping=slot_mapping, positions=positions)
    B = context_lens.numel()
    if not (new_lens.numel() == B and seq_lens.numel() == B and cu_seqlens_q.numel() == B + 1):
        _fail("kv_block_plan: new_lens and seq_lens must have one entry for each request, cu_seqlens_q one more")
    _check_table(what, block_table, B, "block_table", slot_mapping)
    if positions.numel() != slot_mapping.numel():
        _fail("kv_block_plan: positions and slot_mapping differ in length")
    if not (free_begin.numel() == 1 and free_end.numel() == 1 and status.numel() == 3):
        _fail("kv_block_plan: free_begin and free_end must have 1 entry, status 3")
    _C.kv_block_plan(context_lens, new_lens, block_table, free_blocks, free_begin, block_size, num_blocks,
                     slot_mapping, positions, cu_seqlens_q, seq_lens, free_end, status)


def _rotary_embedding_scaled(positions, query, key, inv_freq, attn_factor, is_neox, query_out, key_out):
    what = "rotary_embedding_scaled"
    _check_ints(what, query, torch.int64, positions=positions)
    _check_inv_freq(what, inv_freq, query)
    T = positions.numel()
    _check_heads(what, query, T, "query", query)
    _check_heads(what, query_out, T, "query_out", query)
    if query_out.shape != query.shape:
        _fail("rotary_embedding_scaled: query_out must have the shape of query")
    if (key is None) != (key_out is None):
        _fail("rotary_embedding_scaled: key and key_out come together")
    if key is not None:
        _check_heads(what, key, T, "key", query)
        _check_heads(what, key_out, T, "key_out", query)
        if not (key_out.shape == key.shape and key.shape[2] == query.shape[2]):
            _fail("rotary_embedding_scaled: key_out must have the shape of key, and both the head size of query")
    _C.rope_scaled(positions, query, key, inv_freq, attn_factor, is_neox, query_out, key_out)


def _store_kv_cache_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping, query, positions, inv_freq,
                        attn_factor, is_neox, query_out):
    what = "store_kv_cache_fp8"
    _check_ints(what, key, torch.int64, slot_mapping=slot_mapping)
    T = slot_mapping.numel()
    _check_heads(what, key, T, "key", key)
    _check_heads(what, value, T, "value", key)
    _check_cache(what, k_cache, k_scale, "k", key)
    _check_cache(what, v_cache, v_scale, "v", key)
    if not (value.shape == key.shape and v_cache.shape == k_cache.shape and k_cache.shape[2:] == key.shape[1:]):
        _fail("store_kv_cache_fp8: key and value must have one shape, the caches too, with the same heads")
    if (positions is None) != (inv_freq is None):
        _fail("store_kv_cache_fp8: positions and inv_freq come together")
    if (query is None) != (query_out is None):
        _fail("store_kv_cache_fp8: query and query_out come together")
    if positions is not None:
        _check_ints(what, key, torch.int64, positions=positions)
        _check_inv_freq(what, inv_freq, key)
        if positions.numel() != T:
            _fail("store_kv_cache_fp8: positions and slot_mapping differ in length")
    if query is not None:
        if positions is None:
            _fail("store_kv_cache_fp8: a query is given to be rotated, and needs positions")
        _check_heads(what, query, T, "query", key)
        _check_heads(what, query_out, T, "query_out", key)
        if not (query_out.shape == query.shape and query.shape[2] == key.shape[2]):
            _fail("store_kv_cache_fp8: query_out must have the shape of query, with the head size of key")
    _C.kv_store_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping, query, positions, inv_freq,
                    attn_factor, is_neox, query_out)


def _merge_state_v2(v_a, s_a, v_b, s_b, v_merged, s_merged):
    """sgl-kernel/csrc/attention/merge_attn_states.cu:180-204: contiguous [tokens, heads, D] /
    [tokens, heads] operands on one device."""
    for t in (v_a, s_a, v_b, s_b, v_merged, s_merged):
        _require(t.is_cuda and t.is_contiguous(), "merge_state_v2: contiguous device tensors expected")
    _require(v_a.dim() == 3 and s_a.dim() == 2 and v_b.shape == v_a.shape and s_b.shape == s_a.shape
             and v_merged.shape == v_a.shape and s_merged.shape == s_a.shape
             and s_a.shape == v_a.shape[:2], "merge_state_v2: shape mismatch")
    _require(v_merged.dtype == torch.bfloat16 and v_a.dtype == torch.bfloat16
             and v_b.dtype == torch.bfloat16, "merge_state_v2: bfloat16 states only")
    _require(s_a.dtype == torch.float32 and s_b.dtype == torch.float32
             and s_merged.dtype == torch.float32, "merge_state_v2: float32 log-sum-exps only")
    _C.merge_attn_states(v_merged.unsqueeze(0), s_merged.unsqueeze(0), v_a.unsqueeze(0),
                         s_a.unsqueeze(0), v_b.unsqueeze(0), s_b.unsqueeze(0), lse_layout="bsh")


_IMPLS = {
    "kv_block_plan": _kv_block_plan,
    "rotary_embedding_scaled": _rotary_embedding_scaled,
    "store_kv_cache_fp8": _store_kv_cache_fp8,
    "merge_state_v2": _merge_state_v2,
    "fp8_scaled_mm": _fp8_scaled_mm,
    "fp8_blockwise_scaled_mm": _fp8_blockwise_scaled_mm,
    "sgl_per_token_quant_fp8": _sgl_per_token_quant_fp8,
    "sgl_per_token_group_quant_8bit": _sgl_per_token_group_quant_8bit,
    "sgl_per_tensor_quant_fp8": _sgl_per_tensor_quant_fp8,
    "rmsnorm": _rmsnorm,
    "fused_add_rmsnorm": _fused_add_rmsnorm,
    "rotary_embedding": _rotary_embedding,
    "apply_rope_pos_ids_cos_sin_cache": _apply_rope_pos_ids_cos_sin_cache,
    "fwd": _fwd,
    "fwd_paged_fp8": _fwd_paged_fp8,
}
for _name, _fn in _IMPLS.items():
    _lib.impl(_name, _fn, "CUDA")


# --------------------------------------------------------------- fake (meta) implementations --
@torch.library.register_fake("sgl_kernel::fp8_scaled_mm")
def _fake_fp8_scaled_mm(mat_a, mat_b, scales_a, scales_b, out_dtype, bias):
    return mat_a.new_empty((mat_a.shape[0], mat_b.shape[1]), dtype=out_dtype)


@torch.library.register_fake("sgl_kernel::fp8_blockwise_scaled_mm")
def _fake_fp8_blockwise_scaled_mm(mat_a, mat_b, scales_a, scales_b, out_dtype):
    return mat_a.new_empty((mat_a.shape[0], mat_b.shape[1]), dtype=out_dtype)


def _fake_none(*args, **kwargs):
    return None


for _name in ("sgl_per_token_quant_fp8", "sgl_per_token_group_quant_8bit", "sgl_per_tensor_quant_fp8",
              "rmsnorm", "fused_add_rmsnorm", "rotary_embedding", "apply_rope_pos_ids_cos_sin_cache",
              "merge_state_v2", "kv_block_plan", "rotary_embedding_scaled", "store_kv_cache_fp8"):
    torch.library.register_fake("sgl_kernel::" + _name)(_fake_none)


@torch.library.register_fake("sgl_kernel::fwd_paged_fp8")
def _fake_fwd_paged_fp8(q, *rest, **kw):
    return _fake_fwd(q, None, None, None, None, None, None, None, None)[:2]


@torch.library.register_fake("sgl_kernel::fwd")
def _fake_fwd(q, k, v, k_new, v_new, q_v, out, cu_seqlens_q, cu_seqlens_k, *rest, **kw):
    o = torch.empty_like(q) if out is None else out
    if q.dim() == 4:
        lse = q.new_empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32)
    else:
        lse = q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32)
    e = q.new_empty((0,), dtype=torch.float32)
    return o, lse, e, e
