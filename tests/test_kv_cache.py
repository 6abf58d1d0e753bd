"""The operators around the paged 8-bit KV cache, without a GPU: what their checks refuse (in
Python and at the C ABI, before anything is launched), shapes under tracing, the frequencies of
the long-context scalings, and the oracle of the GPU tests against hand-made cases."""
import ctypes
import math

import pytest
import torch

from sglang_diffusion_amd import _C
from sglang_diffusion_amd.layers.rotary import scaled_inv_freq
from tests import kv_cache_oracle as oracle

FP8 = torch.float8_e4m3fn
BF = torch.bfloat16


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def i64(*shape):
    return torch.zeros(shape, dtype=torch.int64)


def call(name, **kw):
    """The op on CPU tensors: its checks run, then the device is refused."""
    from sgl_kernel import _ops

    return _ops._IMPLS[name](**kw) if name in _ops._IMPLS else getattr(torch.ops.sgl_kernel, name).default(**kw)


def fwd_args(**change):
    B, T, H, Hk, D, blocks, size = 2, 5, 4, 2, 64, 7, 16
    codes = torch.zeros(blocks, size, Hk, D).to(FP8)
    a = dict(q=torch.zeros(T, H, D, dtype=BF), k=codes, v=codes.clone(), k_new=None, v_new=None, q_v=None, out=None,
             cu_seqlens_q=i32(B + 1), cu_seqlens_k=None, cu_seqlens_k_new=None, seqused_q=None, seqused_k=i32(B),
             max_seqlen_q=3, max_seqlen_k=None, page_table=i32(B, 3), kv_batch_idx=None, leftpad_k=None,
             rotary_cos=None, rotary_sin=None, seqlens_rotary=None, q_descale=None,
             k_descale=torch.ones(blocks, Hk), v_descale=torch.ones(blocks, Hk), softmax_scale=None, is_causal=True,
             window_left=-1, window_right=-1, attention_chunk=0, softcap=0.0, is_rotary_interleaved=False,
             scheduler_metadata=None, num_splits=0, pack_gqa=None, sm_margin=0, sinks=None)
    a.update(change)
    return a


def refused(name, args, match):
    with pytest.raises(RuntimeError, match=match):
        call(name, **args)


def test_attend_reaches_the_library_and_no_cpu_form():
    refused("fwd", fwd_args(), "HIP device")
    import sgl_kernel

    a = fwd_args()
    with pytest.raises(RuntimeError, match="HIP device"):
        sgl_kernel.flash_attn_with_kvcache(a["q"], a["k"], a["v"], cache_seqlens=a["seqused_k"], page_table=a["page_table"],
                                           cu_seqlens_q=a["cu_seqlens_q"], max_seqlen_q=3, k_descale=a["k_descale"],
                                           v_descale=a["v_descale"], causal=True)


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(5, 4, 64)), "bfloat16"),
    (dict(q=torch.zeros(5, 4, 128, dtype=BF)), "head size"),
    (dict(q=torch.zeros(5, 3, 64, dtype=BF)), "multiple"),
    (dict(q=torch.zeros(5, 4, 64, 2, dtype=BF)[..., 0]), "contiguous last"),
    (dict(q=torch.zeros(3, 5, 4, 64, dtype=BF), cu_seqlens_q=None), "batched"),
    (dict(q=torch.zeros(2, 5, 4, 64, dtype=BF)), "batched"),
    (dict(v=torch.zeros(7, 16, 2, 64, dtype=BF)), "v_cache"),
    (dict(v=torch.zeros(7, 32, 2, 64).to(FP8)), "one shape"),
    (dict(k_descale=None), "scales of k_cache"),
    (dict(k_descale=torch.ones(2, 2)), "scales of k_cache"),
    (dict(v_descale=torch.ones(7, 2, dtype=torch.float64)), "scales of v_cache"),
    (dict(v_descale=torch.ones(2, 7).t()), "scales of v_cache"),
    (dict(seqused_k=None), "lengths"),
    (dict(seqused_k=i64(2)), "cache_seqlens"),
    (dict(cu_seqlens_q=None), "cu_seqlens_q"),
    (dict(cu_seqlens_q=i32(5)), "disagree"),
    (dict(page_table=i64(2, 3)), "page_table"),
    (dict(page_table=i32(3, 3)), "page_table"),
    (dict(page_table=i32(3, 2).t()), "page_table"),
    (dict(is_causal=False, window_left=5, window_right=0), "sliding"),
    (dict(window_left=5, window_right=2), "sliding"),
    (dict(attention_chunk=16), "attention_chunk"),
    (dict(softcap=5.0), "softcap"),
    (dict(sinks=torch.zeros(4)), "sinks"),
    (dict(k_new=torch.zeros(1)), "k_new"),
    (dict(cu_seqlens_k=i32(3)), "cu_seqlens_k"),
    (dict(out=torch.zeros(5, 4, 64)), "out must match"),
    (dict(out=torch.zeros(5, 4, 64, dtype=BF)), "HIP device"),
])
def test_attend_refuses(change, match):
    refused("fwd", fwd_args(**change), match)


def test_a_16_bit_paged_cache_is_still_refused():
    codes = torch.zeros(7, 16, 2, 64, dtype=BF)
    refused("fwd", fwd_args(k=codes, v=codes, k_descale=None, v_descale=None), "not supported")
    import sgl_kernel

    q = torch.zeros(5, 4, 64, dtype=BF)
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        sgl_kernel.flash_attn_with_kvcache(q, codes, codes, cache_seqlens=i32(2), page_table=i32(2, 3))
    with pytest.raises(RuntimeError, match="page_table"):
        sgl_kernel.flash_attn_with_kvcache(q, codes.to(FP8), codes.to(FP8), cache_seqlens=i32(2))
    with pytest.raises(NotImplementedError):
        sgl_kernel.flash_attn_with_kvcache(q, codes, codes, score_mod=lambda s: s)
    for other in (dict(k=q), dict(v=q), dict(qv=q), dict(rotary_cos=q), dict(rotary_sin=q), dict(cache_batch_idx=i32(2)),
                  dict(cache_leftpad=i32(2)), dict(cu_seqlens_k_new=i32(3)), dict(rotary_seqlens=i32(2)),
                  dict(q_descale=q), dict(sinks=q), dict(attention_chunk=8), dict(softcap=1.0)):
        with pytest.raises(RuntimeError, match="not implemented"):
            sgl_kernel.flash_attn_with_kvcache(q, codes.to(FP8), codes.to(FP8), cache_seqlens=i32(2),
                                               page_table=i32(2, 3), **other)


def plan_args(**change):
    a = dict(context_lens=i32(2), new_lens=i32(2), block_table=i32(2, 4), free_blocks=i32(9), free_begin=i32(1),
             block_size=16, num_blocks=20, slot_mapping=i64(6), positions=i64(6), cu_seqlens_q=i32(3), seq_lens=i32(2),
             free_end=i32(1), status=i32(3))
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    ({}, "HIP device"),
    (dict(context_lens=i64(2)), "context_lens"),
    (dict(new_lens=i32(3)), "one entry for each"),
    (dict(cu_seqlens_q=i32(2)), "one entry for each"),
    (dict(block_table=i32(3, 4)), "block_table"),
    (dict(block_table=i32(4, 2).t()), "block_table"),
    (dict(positions=i64(5)), "differ in length"),
    (dict(slot_mapping=i32(6)), "slot_mapping"),
    (dict(status=i32(2)), "status 3"),
    (dict(free_end=i32(2)), "1 entry"),
])
def test_plan_refuses(change, match):
    refused("kv_block_plan", plan_args(**change), match)


def rope_args(**change):
    a = dict(positions=i64(5), query=torch.zeros(5, 4, 64, dtype=BF), key=torch.zeros(5, 2, 64, dtype=BF),
             inv_freq=torch.ones(16, dtype=torch.float64), attn_factor=1.0, is_neox=True,
             query_out=torch.zeros(5, 4, 64, dtype=BF), key_out=torch.zeros(5, 2, 64, dtype=BF))
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    ({}, "HIP device"),
    (dict(positions=i32(5)), "positions"),
    (dict(positions=i64(4)), "query"),
    (dict(query=torch.zeros(5, 256, dtype=BF)), "query"),
    (dict(query_out=torch.zeros(5, 3, 64, dtype=BF)), "shape of query"),
    (dict(key=None), "together"),
    (dict(key=torch.zeros(5, 2, 32, dtype=BF), key_out=torch.zeros(5, 2, 32, dtype=BF)), "head size"),
    (dict(inv_freq=torch.ones(16, dtype=BF)), "inv_freq"),
    (dict(inv_freq=torch.ones(32, dtype=torch.float64)[::2]), "inv_freq"),
])
def test_rope_refuses(change, match):
    refused("rotary_embedding_scaled", rope_args(**change), match)


def store_args(**change):
    codes = torch.zeros(7, 16, 2, 64).to(FP8)
    a = dict(key=torch.zeros(5, 2, 64, dtype=BF), value=torch.zeros(5, 2, 64, dtype=BF), k_cache=codes,
             v_cache=codes.clone(), k_scale=torch.ones(7, 2), v_scale=torch.ones(7, 2), slot_mapping=i64(5), query=None,
             positions=None, inv_freq=None, attn_factor=1.0, is_neox=True, query_out=None)
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    ({}, "HIP device"),
    (dict(value=torch.zeros(5, 1, 64, dtype=BF)), "one shape"),
    (dict(key=torch.zeros(5, 2, 64)), "key"),
    (dict(slot_mapping=i32(5)), "slot_mapping"),
    (dict(slot_mapping=i64(4)), "key"),
    (dict(k_cache=torch.zeros(7, 16, 2, 64, dtype=BF)), "k_cache"),
    (dict(k_scale=torch.ones(7)), "scales of k_cache"),
    (dict(positions=i64(5)), "together"),
    (dict(positions=i64(4), inv_freq=torch.ones(16)), "differ in length"),
    (dict(query=torch.zeros(5, 4, 64, dtype=BF), query_out=torch.zeros(5, 4, 64, dtype=BF)), "needs positions"),
    (dict(query=torch.zeros(5, 4, 64, dtype=BF)), "together"),
])
def test_store_refuses(change, match):
    refused("store_kv_cache_fp8", store_args(**change), match)


# ----------------------------------------------------------------------------------- C ABI --
def last_error():
    return _C.load_library().mi355_last_error().decode()


def test_c_abi_refuses_before_any_launch():
    """Pointers are never touched on the host: any non-null number stands for one."""
    lib = _C.load_library()
    a = _C.PagedAttnArgs(*([16] * 10), 2, 5, 4, 2, 64, 3, *([64] * 8), *([64] * 6), 3, 3, 7, 16, 0.1, 1, -1, None, 0)
    need = lib.mi355_paged_attn_workspace_bytes(ctypes.byref(a))
    assert need == 0                                     # 48 tokens at most: nothing to split

    def attn(**change):
        b = _C.PagedAttnArgs()
        ctypes.pointer(b)[0] = a
        for name, value in change.items():
            setattr(b, name, value)
        assert lib.mi355_paged_attn_fp8(ctypes.byref(b), None) == -1
        return last_error()

    assert "head size" in attn(D=96)
    assert "shape" in attn(H=5)
    assert "power of two" in attn(block_size=24)
    assert "power of two" in attn(block_size=8)
    assert "power of two" in attn(block_size=2048)
    assert "window" in attn(causal=0, window_left=3)
    assert "null" in attn(q=None)
    assert "null" in attn(page_table=None)
    assert "multiples of 8" in attn(q_ss=60)
    assert "16 bytes" in attn(kc_st=72)
    assert "aligned" in attn(k_cache=24)
    assert "page table" in attn(table_width=1 << 28)
    assert "too large" in attn(kc_st=1 << 24)
    assert "overlap" in attn(o_ss=0) and "overlap" in attn(o_sh=0)
    assert "overlap" in attn(cu_seqlens_q=None, o_sb=0)
    assert "workspace" in attn(table_width=1 << 16, table_stride=1 << 16)
    assert "null args" in (lib.mi355_paged_attn_fp8(None, None), last_error())[1]
    b = _C.PagedAttnArgs()
    ctypes.pointer(b)[0] = a
    b.table_width = 1 << 16
    assert lib.mi355_paged_attn_workspace_bytes(ctypes.byref(b)) > 0
    b.B = 0
    assert lib.mi355_paged_attn_fp8(ctypes.byref(b), None) == 0     # nothing to do

    s = _C.KvStoreArgs(16, 16, 128, 64, 128, 64, 16, 16, 2048, 128, 64, 2048, 128, 64, 16, 16, 16, 5, 2, 64, 16, 7)

    def store(**change):
        b = _C.KvStoreArgs()
        ctypes.pointer(b)[0] = s
        for name, value in change.items():
            setattr(b, name, value)
        assert lib.mi355_kv_store_fp8(ctypes.byref(b), None) == -1
        return last_error()

    assert "head size" in store(D=80)
    assert "power of two" in store(block_size=17)
    assert "null" in store(k=None)
    assert "null" in store(k_scale=None)
    assert "multiples of 8" in store(kc_st=100)
    for name in ("kc_sb", "kc_st", "kc_sh", "vc_sb", "vc_st", "vc_sh"):
        assert "overlap" in store(**{name: 0})
    assert "overlap" in store(Hq=3, q=16, q_out=16, positions=16, inv_freq=16, rot_dim=64, qo_sh=64)
    assert "aligned" in store(v=24)
    assert "queries need" in store(Hq=3, q=16, q_out=16)
    assert "rot_dim" in store(positions=16, inv_freq=16, rot_dim=24)
    assert "rot_dim" in store(positions=16, inv_freq=16, rot_dim=80)
    s.tokens = 0
    assert lib.mi355_kv_store_fp8(ctypes.byref(s), None) == 0

    def rope(D=64, rot=64, st=256, ptr=16, out_st=256):
        rc = lib.mi355_rope_scaled(16, ptr, 16, None, None, 5, 4, 0, D, rot, st, 64, out_st, 64, 0, 0, 0, 0, 16, 1, 1.0,
                                   1, None)
        assert rc == -1
        return last_error()

    assert "rot_dim" in rope(rot=128) and "rot_dim" in rope(rot=40) and "rot_dim" in rope(rot=0)
    assert "head size" in rope(D=264, rot=64) and "head size" in rope(D=60, rot=16)
    assert "multiples of 8" in rope(st=255) and "aligned" in rope(ptr=8) and "overlap" in rope(out_st=0)

    # inputs and outputs 4096 bytes apart, except those named
    names = ["context", "new", "table", "free", "begin", "slots", "positions", "cu", "seq_lens", "free_end", "status"]

    def plan(B=2, block=16, width=4, stride=4, room=6, **at):
        p = {n: at.get(n, 4096 * (i + 1)) for i, n in enumerate(names)}
        rc = lib.mi355_kv_block_plan(p["context"], p["new"], B, p["table"], stride, width, p["free"], 9, p["begin"], block,
                                     20, p["slots"], p["positions"], room, p["cu"], p["seq_lens"], p["free_end"],
                                     p["status"], None)
        assert rc == -1
        return last_error()

    assert "at most" in plan(B=4097) and "power of two" in plan(block=48)
    assert "bad size" in plan(stride=3) and "bad size" in plan(room=1 << 31) and "bad size" in plan(width=1 << 27)
    assert "null" in plan(cu=None) and "null" in plan(slots=None) and "null" in plan(table=None)
    for out, size in (("slots", 48), ("positions", 48), ("cu", 12), ("seq_lens", 8), ("free_end", 4), ("status", 12)):
        for n in names:
            if n != out:
                assert "share memory" in plan(**{out: 4096 * (names.index(n) + 1)})
        assert "share memory" in plan(**{out: 4096 - size + 4})       # the context's first length
    assert "share memory" in plan(free=4096 * 3 + 28)                 # the table's last entry


def test_shapes_under_tracing():
    a = fwd_args()
    meta = {k: v.to("meta") if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    out, lse, *_ = torch.ops.sgl_kernel.fwd(**meta)
    assert out.shape == (5, 4, 64) and lse.shape == (4, 5) and lse.dtype == torch.float32
    same = [meta[n] for n in ("q", "k", "v", "k_descale", "v_descale", "page_table", "seqused_k", "cu_seqlens_q")]
    out, lse = torch.ops.sgl_kernel.fwd_paged_fp8(*same, 3, None, True, -1, -1)
    assert out.shape == (5, 4, 64) and lse.shape == (4, 5)
    assert torch.ops.sgl_kernel.fwd_paged_fp8_out(*same, 3, None, True, -1, -1, torch.empty_like(same[0])).shape == (4, 5)
    meta["q"] = torch.empty(2, 3, 4, 64, dtype=BF, device="meta")
    out, lse, *_ = torch.ops.sgl_kernel.fwd(**meta)
    assert out.shape == (2, 3, 4, 64) and lse.shape == (2, 4, 3)
    for name, args in (("kv_block_plan", plan_args()), ("rotary_embedding_scaled", rope_args()),
                       ("store_kv_cache_fp8", store_args())):
        op = getattr(torch.ops.sgl_kernel, name)
        assert op(**{k: v.to("meta") if isinstance(v, torch.Tensor) else v for k, v in args.items()}) is None


# ----------------------------------------------------------------------------- frequencies --
def test_scaled_frequencies():
    f, factor = scaled_inv_freq(64, 10000.0)
    assert factor == 1.0 and f.dtype == torch.float64 and f.shape == (32,)
    assert torch.allclose(f, 1.0 / 10000.0 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 64), rtol=1e-14)
    g, factor = scaled_inv_freq(64, 10000.0, {"rope_type": "linear", "factor": 8.0})
    assert factor == 1.0 and torch.equal(g, f / 8.0)

    cfg = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
           "original_max_position_embeddings": 8192}
    f, _ = scaled_inv_freq(128, 500000.0)
    g, factor = scaled_inv_freq(128, 500000.0, cfg)
    wave = 2 * math.pi / f
    assert factor == 1.0
    assert torch.equal(g[wave < 8192 / 4.0], f[wave < 8192 / 4.0])
    assert torch.allclose(g[wave > 8192 / 1.0], f[wave > 8192 / 1.0] / 8.0, rtol=1e-15)
    mid = (wave >= 8192 / 4.0) & (wave <= 8192)
    smooth = (8192 / wave[mid] - 1.0) / 3.0
    assert mid.any() and torch.allclose(g[mid], (1 - smooth) * f[mid] / 8.0 + smooth * f[mid], rtol=1e-13)

    cfg = {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    f, _ = scaled_inv_freq(128, 10000.0)
    g, factor = scaled_inv_freq(128, 10000.0, cfg)
    turns = 4096 * f / (2 * math.pi)
    assert factor == pytest.approx(0.1 * math.log(16.0) + 1.0)
    assert torch.equal(g[turns > 40], f[turns > 40])                 # the fast pairs as they were
    assert torch.allclose(g[turns < 0.8], f[turns < 0.8] / 16.0, rtol=1e-15)
    assert ((g <= f) & (g >= f / 16.0 * (1 - 1e-15))).all() and (g[1:] < g[:-1]).all()
    assert scaled_inv_freq(128, 10000.0, dict(cfg, attention_factor=1.25))[1] == 1.25
    with pytest.raises(ValueError):
        scaled_inv_freq(63)
    with pytest.raises(ValueError):
        scaled_inv_freq(64, scaling={"rope_type": "unheard of"})


# ---------------------------------------------------------------------------------- oracle --
def test_oracle_of_the_plan_by_hand():
    got = oracle.plan([0, 15, 16], [2, 2, 1], [[-1, -1], [4, -1], [6, -1]], [9, 8, 7, 5], 1, 16, 10, 7)
    table, slots, positions, cu, lens, end, status = got
    assert table == [[8, -1], [4, 7], [6, 5]] and status == [0, 0, 0] and end == 4
    assert slots == [128, 129, 4 * 16 + 15, 7 * 16, 5 * 16, -1, -1]
    assert positions == [0, 1, 15, 16, 16, 0, 0] and cu == [0, 2, 4, 5] and lens == [2, 17, 17]


def test_oracle_rounding_is_that_of_torch():
    v = torch.cat([torch.linspace(-448, 448, 4001), torch.linspace(-0.04, 0.04, 4001), torch.tensor([464.0, -1e9])]).float()
    assert torch.equal(oracle.e4m3(v.double()), v.clamp(-448, 448).to(FP8).double())
    assert torch.isnan(oracle.e4m3(torch.tensor([math.inf, math.nan], dtype=torch.float64))).all()


def test_oracle_of_the_attention_is_softmax():
    """One sequence in two blocks, no masks but the causal one: torch's own softmax in 64 bits."""
    g = torch.Generator().manual_seed(0)
    codes = [(torch.randn(3, 16, 1, 64, generator=g) * 50).to(FP8).float() for _ in range(2)]
    scales = [torch.rand(3, 1, generator=g) * 0.01 for _ in range(2)]
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    q = torch.randn(4, 2, 64, generator=g)
    out, lse, _ = oracle.attend(q, *codes, *scales, table, [20], [0, 4], 0.125, True, -1)
    k, v = ((torch.cat([c[2], c[0]]).double() * torch.cat([s[2].expand(16), s[0].expand(16)]).double()[:, None, None])[:20, 0]
            for c, s in zip(codes, scales))
    for h in range(2):
        s = q[:, h].double() @ k.t() * 0.125
        s = s.masked_fill(torch.arange(20)[None] > torch.arange(16, 20)[:, None], -math.inf)
        assert torch.allclose(out[:, h], torch.softmax(s, -1) @ v, rtol=1e-12)
        assert torch.allclose(lse[h], torch.logsumexp(s, -1), rtol=1e-12)
