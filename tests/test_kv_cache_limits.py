"""Limits of the arguments of the paged attention at the C ABI, before any launch (pointers are never
touched on the host, any number stands for one)."""
import ctypes

from sglang_diffusion_amd import _C
from tests.test_kv_cache_overlap import D, H, HK, K, Q, QO, T, V


def args(**change):
    a = _C.PagedAttnArgs(q=Q, out=QO, k_cache=K, v_cache=V, k_scale=16, v_scale=16, cu_seqlens_q=16, cache_seqlens=16,
                         page_table=16, B=2, Sq=T, H=H, Hk=HK, D=D, max_seqlen_q=3, q_sb=0, q_ss=H * D, q_sh=D, o_sb=0,
                         o_ss=H * D, o_sh=D, kc_sb=2048, kc_st=128, kc_sh=64, vc_sb=2048, vc_st=128, vc_sh=64,
                         table_stride=3, table_width=3, num_blocks=7, block_size=16, softmax_scale=0.1, causal=1,
                         window_left=-1)
    for name, value in change.items():
        setattr(a, name, value)
    return a


def workspace(**change):
    lib = _C.load_library()
    need = lib.mi355_paged_attn_workspace_bytes(ctypes.byref(args(**change)))
    return need, lib.mi355_last_error().decode()


def test_rows_whose_number_does_not_fit_64_bits():
    """2^61 rows, and 2^65 and 2^64, which are none in 64 bits."""
    for B, Sq, heads in ((1 << 20, 1 << 28, 1 << 13), (1 << 23, 1 << 30, 1 << 12), (1 << 22, 1 << 30, 1 << 12)):
        need, message = workspace(cu_seqlens_q=None, B=B, Sq=Sq, H=heads, Hk=1)
        assert need == -1 and "too many rows" in message


def test_windows():
    need, message = workspace(causal=0, window_left=3)
    assert need == -1 and "causal" in message
    wide = dict(table_width=1 << 16, table_stride=1 << 16)
    want, _ = workspace(**wide)
    assert want > 0
    for window in (1 << 20, 1 << 40, (1 << 62) + 1, (1 << 63) - 1):                # none of them hides a key
        assert workspace(window_left=window, **wide)[0] == want
    assert workspace(window_left=0, **wide)[0] == 0                                # a tile of keys is not split
