"""Rotary embeddings of the DiT path.

NDRotaryEmbedding.forward_uncached mirrors python/sglang/multimodal_gen/runtime/layers/
rotary_embedding/mrope.py:96-125,259-294 (float64 frequency table, built once per shape on
the host: it is a [S, 64] table, not per-step work); apply_flashinfer_rope_qk_inplace mirrors
rotary_embedding/utils.py:42-121 and runs the fused HIP kernel.
"""
from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch

from .. import _C


class NDRotaryEmbedding(torch.nn.Module):
    def __init__(self, rope_dim_list: List[int], rope_theta: float, use_real: bool = False,
                 repeat_interleave_real: bool = False, dtype: torch.dtype = torch.float64):
        super().__init__()
        if use_real or repeat_interleave_real:
            raise NotImplementedError("the Flux path uses use_real=False")
        self.rope_dim_list = rope_dim_list
        self.rope_theta = rope_theta
        self.dtype = dtype

    def forward_uncached(self, pos: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """pos [num_tokens, ndim] -> cos, sin [num_tokens, sum(dims)/2] fp32.  Per axis:
        freqs = 1/theta^(arange(0,dim,2)/dim) in self.dtype, outer(pos, freqs), cos/sin cast
        to fp32 (mrope.py:96-125)."""
        cos_parts, sin_parts = [], []
        for i, dim in enumerate(self.rope_dim_list):
            pos_i = pos[:, i].to(self.dtype)
            freqs = 1.0 / (self.rope_theta ** (
                torch.arange(0, dim, 2, dtype=self.dtype, device=pos.device)[: dim // 2] / dim))
            f = torch.outer(pos_i, freqs)
            cos_parts.append(f.cos().float())
            sin_parts.append(f.sin().float())
        return torch.cat(cos_parts, dim=1).float(), torch.cat(sin_parts, dim=1).float()

    def forward(self, positions: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        return self.forward_uncached(positions)


def apply_flashinfer_rope_qk_inplace(q: torch.Tensor, k: torch.Tensor,
                                     cos_sin_cache: torch.Tensor, *,
                                     head_size: Optional[int] = None, is_neox: bool = False,
                                     positions: Optional[torch.Tensor] = None,
                                     round_cos_sin_to_input_dtype: bool = False):
    """utils.py:42-121.  q,k [bsz, seqlen, nheads, head_size]; cos_sin_cache [seqlen, D] =
    cos | sin (fp32).  `round_cos_sin_to_input_dtype=True` reproduces the reference's
    non-flashinfer fallback, which casts cos/sin to q.dtype first (utils.py:80-83)."""
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("Expected q/k to be 4D [bsz, seqlen, nheads, head_size], "
                         f"got q:{tuple(q.shape)} k:{tuple(k.shape)}")
    if q.shape != k.shape:
        raise ValueError(f"q and k must have the same shape, got {q.shape} vs {k.shape}")
    if not (isinstance(cos_sin_cache, torch.Tensor) and cos_sin_cache.dim() == 2):
        raise ValueError("cos_sin_cache must be a 2D torch.Tensor")
    bsz, seqlen, nheads, d = q.shape
    if head_size is None:
        head_size = d
    if head_size != d:
        raise ValueError(f"head_size mismatch: inferred {d}, but head_size={head_size}")
    half = cos_sin_cache.shape[-1] // 2
    if positions is not None:
        if positions.dtype != torch.long or positions.dim() != 1:
            raise ValueError("positions must be a 1D torch.long Tensor")
        if positions.numel() != bsz * seqlen:
            raise ValueError(f"positions length must be bsz*seqlen={bsz * seqlen}, "
                             f"got {positions.numel()}")
        qf, kf = q.reshape(bsz * seqlen, nheads * d), k.reshape(bsz * seqlen, nheads * d)
        cache = cos_sin_cache.float().contiguous()
        _C.rotary_embedding(positions, qf, kf, d, cache, is_neox)
        return qf.view(bsz, seqlen, nheads, d), kf.view(bsz, seqlen, nheads, d)
    cos = cos_sin_cache[:seqlen, :half]
    sin = cos_sin_cache[:seqlen, half:]
    if round_cos_sin_to_input_dtype:
        cos, sin = cos.to(q.dtype), sin.to(q.dtype)
    cos, sin = cos.float().contiguous(), sin.float().contiguous()
    if q.stride() != k.stride() or q.stride(-1) != 1:
        q, k = q.contiguous(), k.contiguous()
    _C.qk_norm_rope(q, k, None, None, None, None, 0, 0.0, cos, sin, not is_neox)
    return q, k


# what each rope_type of `scaled_inv_freq` uses
_ROPE_KEYS = {
    "default": (),
    "linear": ("factor",),
    "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
    "yarn": ("factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "truncate", "attention_factor",
             "mscale", "mscale_all_dim"),
}


def scaled_inv_freq(rot_dim: int, base: float = 10000.0, scaling: Optional[dict] = None,
                    device=None) -> Tuple[torch.Tensor, float]:
    """Frequencies base^(-2i / rot_dim) in float64, scaled for contexts longer than the trained one,
    and the factor on cosine and sine that goes with them: the `inv_freq` and `attn_factor` of
    `sgl_kernel.rotary_embedding_scaled` and `store_kv_cache_fp8`.  `scaling` is the `rope_scaling`
    entry of a model's config, with its names:

    * {"rope_type": "linear", "factor": f}: all frequencies divided by f.
    * {"rope_type": "llama3", "factor", "low_freq_factor", "high_freq_factor",
      "original_max_position_embeddings"}: pairs that turn fewer than low_freq_factor times over the
      trained length divided by f, those above high_freq_factor kept, the share between
      interpolated over the number of turns.
    * {"rope_type": "yarn", "factor", "original_max_position_embeddings", "beta_fast" (32),
      "beta_slow" (1), "truncate" (True), "attention_factor", "mscale", "mscale_all_dim"}: a ramp over
      the pair index between the pairs that turn beta_fast and beta_slow times, whole indices unless
      truncate is false; attention_factor defaults to m(mscale) / m(mscale_all_dim) with
      m(x) = 0.1 x ln f + 1, and to m(1) without those two.

    A key that the type has no use for raises, since leaving it out may be wrong for the model."""
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError(f"rot_dim must be positive and even, got {rot_dim}")
    freq = base ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    attn_factor = 1.0
    scaling = dict(scaling or {})
    kind = scaling.pop("rope_type", None)
    legacy = scaling.pop("type", None)
    if kind is not None and legacy is not None and kind != legacy:
        raise ValueError(f"rope_type {kind!r} and type {legacy!r} differ")
    kind = kind or legacy or "default"
    if kind not in _ROPE_KEYS:
        raise ValueError(f"unknown rope_type {kind!r}")
    unused = sorted(set(scaling) - set(_ROPE_KEYS[kind]))
    if unused:
        raise ValueError(f"rope_type {kind!r} does not use {unused}: not implemented")
    if kind == "linear":
        freq = freq / scaling["factor"]
    elif kind == "llama3":
        turns = scaling["original_max_position_embeddings"] * freq / (2 * math.pi)
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        if not low < high:
            raise ValueError(f"low_freq_factor {low} must be below high_freq_factor {high}")
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / scaling["factor"])
    elif kind == "yarn":
        trained, factor = scaling["original_max_position_embeddings"], scaling["factor"]

        def given(name, otherwise):
            value = scaling.get(name)
            return otherwise if value is None else value

        def pair_that_turns(times):
            return rot_dim * math.log(trained / (times * 2 * math.pi)) / (2 * math.log(base))

        first, last = pair_that_turns(given("beta_fast", 32)), pair_that_turns(given("beta_slow", 1))
        if given("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rot_dim - 1)
        ramp = (torch.arange(rot_dim // 2, dtype=torch.float64) - first) / (max(last - first, 0.001))
        keep = 1.0 - ramp.clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)

        def growth(x):
            return 0.1 * x * math.log(factor) + 1.0 if factor > 1 else 1.0

        attn_factor = scaling.get("attention_factor")
        scales = [scaling.get("mscale"), scaling.get("mscale_all_dim")]
        if attn_factor is None:
            if (scales[0] is None) != (scales[1] is None) or 0 in scales:
                raise ValueError("mscale and mscale_all_dim come together and are not 0 (or attention_factor is given)")
            attn_factor = growth(1.0) if scales[0] is None else growth(scales[0]) / growth(scales[1])
    return freq.to(device), float(attn_factor)
