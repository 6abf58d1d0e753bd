"""Layouts in which rows of one tensor lie between those of another without touching them are taken, in
place, by the operators around the paged 8-bit KV cache; the same ones shifted are refused.  Bit for bit
what the operators give on tensors of their own."""
import pytest
import torch

from tests.test_kv_cache_gpu import DEV, Case, empty_cache

pytestmark = pytest.mark.gpu


def projections(T, H, Hk, D):
    """(name, q, k, v) as views: heads side by side, heads outside tokens, q / k / v of a head side by side."""
    wide = torch.randn(T, (H + 2 * Hk) * D, device=DEV).bfloat16()
    yield "fused", *(wide[:, a * D:b * D].view(T, b - a, D) for a, b in ((0, H), (H, H + Hk), (H + Hk, H + 2 * Hk)))
    heads = torch.randn(H + 2 * Hk, T, D, device=DEV).bfloat16().permute(1, 0, 2)
    yield "head by head", heads[:, :H], heads[:, H:H + Hk], heads[:, H + Hk:]
    if H == Hk:
        inner = torch.randn(T, H, 3, D, device=DEV).bfloat16()
        yield "in each head", inner[:, :, 0], inner[:, :, 1], inner[:, :, 2]
        outer = torch.randn(H, 3, T, D, device=DEV).bfloat16().permute(1, 2, 0, 3)
        yield "in each head, heads outside", outer[0], outer[1], outer[2]


@pytest.mark.parametrize("T,H,Hk", [(1, 4, 2), (33, 4, 2), (20, 3, 3), (1, 1, 1), (9000, 2, 2)])
def test_rope_and_store_in_place(device, T, H, Hk):
    import sgl_kernel

    D, block = 64, 16
    f = (10000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32)).to(DEV)
    positions = torch.arange(T, device=DEV) + 3
    slots = torch.arange(T, device=DEV)
    for name, q, k, v in projections(T, H, Hk, D):
        own = [x.contiguous().clone() for x in (q, k, v)]
        sgl_kernel.rotary_embedding_scaled(positions, own[0], own[1], f)
        blocks = -(-T // block)
        (kc, ks), (vc, vs) = empty_cache(blocks, block, Hk, D, 1), empty_cache(blocks, block, Hk, D, 2)
        both = [x.clone() for x in (kc, vc, ks, vs)]
        before = k.contiguous().clone()
        sgl_kernel.store_kv_cache_fp8(k, v, kc, vc, ks, vs, slots, q, positions, f)      # q in place
        assert torch.equal(q, own[0]) and torch.equal(k, before) and torch.equal(v, own[2]), name
        sgl_kernel.store_kv_cache_fp8(own[1], own[2], *both, slots)
        for a, b in zip((kc, vc, ks, vs), both):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name
        sgl_kernel.rotary_embedding_scaled(positions, k, None, f)
        assert torch.equal(k, own[1]) and torch.equal(v, own[2]), name
        # queries and keys at once, turned back
        sgl_kernel.rotary_embedding_scaled(-positions, q, k, f)
        sgl_kernel.rotary_embedding_scaled(-positions, own[0], own[1], f)
        assert torch.equal(q, own[0]) and torch.equal(k, own[1]), name


def test_caches_in_one_buffer(device):
    """Keys and values of a block side by side, of a token, and of a head."""
    import sgl_kernel

    T, Hk, D, block, blocks = 40, 2, 64, 16, 4
    k, v = (torch.randn(T, Hk, D, device=DEV).bfloat16() for _ in range(2))
    slots = torch.arange(T, device=DEV) + 5
    want = None
    for shape, at in (((blocks, 2, block, Hk, D), 1), ((blocks, block, 2, Hk, D), 2), ((blocks, block, Hk, 2, D), 3),
                      ((2, blocks, block, Hk, D), 0)):
        pool = torch.zeros(shape, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
        kc, vc = pool.unbind(at)
        scales = [torch.ones(blocks, Hk, device=DEV) for _ in range(2)]
        sgl_kernel.store_kv_cache_fp8(k, v, kc, vc, *scales, slots)
        got = [x.contiguous().view(torch.uint8) for x in (kc, vc)] + scales
        assert want is None or all(torch.equal(a, b) for a, b in zip(got, want)), shape
        want = got
        with pytest.raises(RuntimeError, match="overlap"):
            sgl_kernel.store_kv_cache_fp8(k, v, kc, kc, *scales, slots)
        with pytest.raises(RuntimeError, match="overlap"):
            sgl_kernel.store_kv_cache_fp8(k, v, kc, vc, scales[0], scales[0], slots)


def test_refused(device):
    import sgl_kernel

    T, H, Hk, D = 12, 4, 2, 64
    f = torch.ones(32, dtype=torch.float64, device=DEV)
    positions = torch.arange(T, device=DEV)
    pool = torch.randn(3 * T, H, D, device=DEV).bfloat16()
    keep = pool.clone()
    q, k = pool[:T], pool[2 * T:, :Hk]
    with pytest.raises(RuntimeError, match="overlaps its input"):
        sgl_kernel.rotary_embedding_scaled(positions, q, None, f, query_out=pool[1:T + 1])
    with pytest.raises(RuntimeError, match="the other tensor"):
        sgl_kernel.rotary_embedding_scaled(positions, q, k, f, query_out=pool[T + 1:2 * T + 1])
    kc, ks = empty_cache(2, 16, Hk, D, 1)
    vc, vs = empty_cache(2, 16, Hk, D, 2)
    with pytest.raises(RuntimeError, match="overlaps keys, values or queries"):
        sgl_kernel.store_kv_cache_fp8(k, k, kc, vc, ks, vs, positions, q, positions, f, query_out=pool[T + 1:2 * T + 1])
    assert torch.equal(pool, keep)

    c = Case([3, 2], [40, 30], H, Hk, D, 16, 70)
    wide = torch.randn(6, H, D, device=DEV).bfloat16()
    wide[:5] = c.q.to(DEV)
    want, lse = c.check()

    def fwd(q, out):
        return torch.ops.sgl_kernel.fwd_paged_fp8_out(q, *c.dev, c.scales[0].to(DEV), c.scales[1].to(DEV), c.table.to(DEV),
                                                      torch.tensor(c.lens, dtype=torch.int32, device=DEV),
                                                      torch.tensor(c.cu, dtype=torch.int32, device=DEV), 3, None, True, -1,
                                                      -1, out)

    for out in (wide[1:], wide[:5].view(H, 5, D).transpose(0, 1), torch.empty(1, H, D, device=DEV).bfloat16().expand(5, -1, -1)):
        with pytest.raises(RuntimeError, match="overlap"):
            fwd(wide[:5], out)
    halves = torch.zeros(5, H, 2, D, device=DEV).bfloat16()               # rows of out between those of q
    halves[:, :, 0] = c.q.to(DEV)
    assert torch.equal(fwd(halves[:, :, 0], halves[:, :, 1]), lse) and torch.equal(halves[:, :, 1], want)
