"""Outputs of the operators around the paged 8-bit KV cache that share memory with inputs or with each
other: refused at the C ABI before any launch (pointers are never touched on the host, any number stands
for one)."""
import ctypes

from sglang_diffusion_amd import _C

T, H, HK, D = 5, 4, 2, 64
Q, K, V, QO, KO = (1 << 20) * 1, (1 << 20) * 2, (1 << 20) * 3, (1 << 20) * 4, (1 << 20) * 5


def error():
    return _C.load_library().mi355_last_error().decode()


def rope(q=Q, q_out=QO, k=K, k_out=KO, q_s=(H * D, D), k_s=(HK * D, D), qo_s=(H * D, D), ko_s=(HK * D, D), tokens=T):
    lib = _C.load_library()
    assert lib.mi355_rope_scaled(16, q, q_out, k, k_out, tokens, H, HK, D, D, *q_s, *qo_s, *k_s, *ko_s, 16, 1, 1.0, 1,
                                 None) == -1
    return error()


def test_rope():
    assert "rows of an output overlap" in rope(qo_s=(D, D))
    assert "rows of an output overlap" in rope(ko_s=(D, T * D - 8))          # heads outside tokens, eight short
    assert "overlaps its input" in rope(q_out=Q, qo_s=(2 * H * D, D))         # the input's pointer, other strides
    assert "overlaps its input" in rope(q_out=Q + 2 * D)                      # shifted by a head
    assert "overlaps its input" in rope(q_out=Q + 2 * H * D * (T - 1) + 16)   # only the last rows meet
    assert "overlaps its input" in rope(k_out=K, ko_s=(D, T * D))
    assert "the other tensor" in rope(q_out=K)
    assert "the other tensor" in rope(k_out=Q)
    assert "the other tensor" in rope(q_out=KO, k_out=KO)
    assert "the other tensor" in rope(q_out=Q, k=Q, k_out=KO)                 # in place, and the keys are queries
    # slices of one projection, the keys' one head too far to the front
    wide = (H + 2 * HK) * D
    assert "the other tensor" in rope(q_out=Q, k=Q + 2 * (H - 1) * D, k_out=KO, q_s=(wide, D), qo_s=(wide, D), k_s=(wide, D))


def store(**change):
    lib = _C.load_library()
    size = 16
    s = _C.KvStoreArgs(k=K, v=V, k_st=HK * D, k_sh=D, v_st=HK * D, v_sh=D, k_cache=Q << 4, v_cache=Q << 5,
                       kc_sb=size * HK * D, kc_st=HK * D, kc_sh=D, vc_sb=size * HK * D, vc_st=HK * D, vc_sh=D,
                       k_scale=Q << 6, v_scale=Q << 7, slot_mapping=16, tokens=T, Hk=HK, D=D, block_size=size, num_blocks=7,
                       positions=16, inv_freq=16, rot_dim=D, inv_freq_is_f64=1, is_neox=1, attn_factor=1.0, Hq=H, q=Q,
                       q_out=QO, q_st=H * D, q_sh=D, qo_st=H * D, qo_sh=D)
    for name, value in change.items():
        setattr(s, name, value)
    assert lib.mi355_kv_store_fp8(ctypes.byref(s), None) == -1
    return error()


def test_store():
    assert "rows of an output overlap" in store(qo_st=D)
    assert "rows of an output overlap" in store(kc_st=D)                      # the second head on the next token
    assert "rows of an output overlap" in store(kc_sb=8 * HK * D)             # blocks half over each other
    assert "rows of an output overlap" in store(vc_sh=D // 2)
    for name in ("K", "V"):
        assert "queries' output overlaps" in store(q_out=globals()[name])
        assert "queries' output overlaps" in store(q_out=globals()[name] + 2 * (HK * D * (T - 1)))
    assert "queries' output overlaps" in store(q_out=Q, qo_st=2 * H * D)
    assert "queries' output overlaps" in store(q_out=Q + 16)
    assert "caches or their scales overlap" in store(v_cache=Q << 4)
    assert "caches or their scales overlap" in store(v_cache=(Q << 4) + 64)   # the next head of the keys
    assert "caches or their scales overlap" in store(v_scale=(Q << 6) + 4 * 7 * HK - 4)


def attend(**change):
    lib = _C.load_library()
    a = _C.PagedAttnArgs(q=Q, out=QO, k_cache=K, v_cache=V, k_scale=16, v_scale=16, cu_seqlens_q=16, cache_seqlens=16,
                         page_table=16, B=2, Sq=T, H=H, Hk=HK, D=D, max_seqlen_q=3, q_sb=0, q_ss=H * D, q_sh=D, o_sb=0,
                         o_ss=H * D, o_sh=D, kc_sb=2048, kc_st=128, kc_sh=64, vc_sb=2048, vc_st=128, vc_sh=64,
                         table_stride=3, table_width=3, num_blocks=7, block_size=16, softmax_scale=0.1, causal=1,
                         window_left=-1)
    for name, value in change.items():
        setattr(a, name, value)
    assert lib.mi355_paged_attn_fp8(ctypes.byref(a), None) == -1
    return error()


def test_attend():
    assert "rows of out overlap" in attend(o_ss=D)
    assert "rows of out overlap" in attend(o_sh=2 * D, o_ss=3 * D)
    assert "rows of out overlap" in attend(cu_seqlens_q=None, o_sb=H * D)
    assert "out overlaps q" in attend(out=Q + 2 * D)
    assert "out overlaps q" in attend(out=Q, o_ss=2 * H * D)
    assert "out overlaps q" in attend(out=Q, o_ss=D, o_sh=T * D)
    assert "out overlaps q" in attend(out=Q + 2 * H * D * (T - 1))
