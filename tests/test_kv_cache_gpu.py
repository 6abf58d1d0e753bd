"""The operators around a paged 8-bit KV cache against plain 64-bit forms (kv_cache_oracle.py):
block tables and slot maps, rotary positions from scaled frequencies, the quantising store, the
attention that reads the cache, and a run of all four as a model step uses them.

Tolerances, derived from the formulas (u = half a step of the type, relative: bf16 2^-8, half
2^-11, fp32 2^-24):
  rope    one rounding to bf16, cosine and sine off by at most 4e-7 (reduced angle 1e-7, Taylor
          sums 2e-9 and their fp32 roundings), two fp32 roundings of the products:
          2^-8 |x| + 1e-6 f (|a| + |z|); and where the angle is large, its own rounding in fp64,
          once here and three times in the kernel (the frequency in quarter turns is a rounded
          product of two rounded numbers, and is multiplied once more): 2^-51 |position * frequency|
  store   codes and scales are exact: one rounding of an exact product with a power of two
  attend  weights rounded to half (2^-11) with scores off by at most 128 u Σ|q k| scale, below
          2e-4 for the sizes here; one rounding to bf16; weights below 2^-14 of the reference are
          off by 2^-25 each:  2^-8 |o| + 8e-4 Σ p |v| + keys 2^-25 max |v|; log-sum-exp 4e-4"""
import math

import pytest
import torch

from tests import kv_cache_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP8 = torch.float8_e4m3fn


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------ plan --
def run_plan(context, new, table, free, begin, block, num_blocks, room):
    import sgl_kernel

    B = len(context)
    width = len(table[0]) if table else 3
    t = i32(table) if table else torch.empty((0, width), dtype=torch.int32, device=DEV)
    outs = dict(slot_mapping=torch.full((room,), 77, dtype=torch.int64, device=DEV),
                positions=torch.full((room,), 77, dtype=torch.int64, device=DEV),
                cu_seqlens_q=i32([77] * (B + 1)), seq_lens=i32([77] * B), free_end=i32([77]),
                status=i32([77] * 3))
    sgl_kernel.kv_block_plan(i32(context), i32(new), t, i32(free), i32([begin]), block, num_blocks, **outs)
    got = (t.tolist(), outs["slot_mapping"].tolist(), outs["positions"].tolist(), outs["cu_seqlens_q"].tolist(),
           outs["seq_lens"].tolist(), outs["free_end"].item(), outs["status"].tolist())
    want = oracle.plan(context, new, table, free, begin, block, num_blocks, room)
    for name, g, w in zip(("table", "slots", "positions", "cu", "seq_lens", "free_end", "status"), got, want):
        assert g == w, name
    return got


def make_plan(B, block, new_hi, ctx_hi, seed, room=7, spare=3, begin=2):
    g = torch.Generator().manual_seed(seed)
    context = torch.randint(0, ctx_hi + 1, (B,), generator=g).tolist()
    new = torch.randint(0, new_hi + 1, (B,), generator=g).tolist()
    held = [-(-c // block) for c in context]
    need = [-(-(c + n) // block) for c, n in zip(context, new)]
    order = torch.randperm(sum(need) + spare + begin, generator=g).tolist()
    width = max(need + [1])
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-1] * (width - h))
        at += h
    return context, new, table, order[at:], begin, block, sum(need) + spare + begin, sum(new) + room


@pytest.mark.parametrize("B,block,new_hi,ctx_hi", [(1, 16, 1, 40), (5, 16, 1, 100), (64, 32, 3, 500), (3, 64, 900, 0),
                                                   (257, 16, 20, 60), (700, 128, 9, 300), (1500, 16, 2, 5),
                                                   (4096, 16, 3, 40)])
def test_plan(device, B, block, new_hi, ctx_hi):
    got = run_plan(*make_plan(B, block, new_hi, ctx_hi, B))
    assert got[-1] == [0, 0, 0]


def test_plan_with_nothing_to_do(device):
    run_plan([], [], [], [4, 5], 1, 16, 8, 3)            # no requests
    run_plan([], [], [], [], 0, 16, 8, 0)                # and no room
    run_plan([5, 16, 0], [0, 0, 0], [[1], [2], [-1]], [3], 0, 16, 8, 4)
    run_plan([5], [-3], [[1]], [3], 0, 16, 8, 4)         # negative lengths count as none
    run_plan([-5], [3], [[1]], [3], 0, 16, 8, 4)


@pytest.mark.parametrize("block", [16, 1024])
def test_plan_at_the_edges_of_blocks(device, block):
    """Contexts and ends on, before and behind the border of a block."""
    ctx = [0, 0, 0, 1, block - 1, block - 1, block, block, block + 1, 2 * block]
    new = [block - 1, block, block + 1, block, 1, 2, 1, block, block - 1, 0]
    held = [-(-c // block) for c in ctx]
    table, at = [], 0
    for h in held:
        table.append([100 + at + i for i in range(h)] + [-1] * (3 - h))
        at += h
    run_plan(ctx, new, table, list(range(40)), 3, block, 200, sum(new) + 1)


def test_plan_gives_nothing_when_something_is_lacking(device):
    args = list(make_plan(9, 16, 40, 100, 3))
    short = args[:]
    short[3] = args[3][:-6]                              # too few free blocks
    assert run_plan(*short)[-1][0] > 0
    room = args[:]
    room[7] = args[7] - 8                                # one token too many
    assert run_plan(*room)[-1] == [0, 1, 0]
    wide = args[:]
    wide[2] = [r[:-1] for r in args[2]]                  # the longest request outgrows its row
    assert run_plan(*wide)[-1][2] >= 1
    huge = args[:]
    huge[1] = [2 ** 31 - 1] * 9                          # lengths that no pool holds
    assert run_plan(*huge)[-1][2] == 9


def test_plan_skips_entries_outside_the_pool(device):
    got = run_plan([20, 3], [4, 4], [[5, 900, -1], [-7, -1, -1]], [1, 2, 3], 0, 16, 64, 9)
    assert got[1][:8] == [-1] * 8


# ------------------------------------------------------------------------------------ rope --
def check_rope(x, got, positions, inv_freq, factor, neox):
    positions = positions.cpu()
    want = oracle.rotate(x, positions, inv_freq, factor, neox)
    size = oracle.rotate(x.abs(), torch.zeros_like(positions), inv_freq, 1.0, neox)
    half = inv_freq.numel()
    if neox:
        pair = size[..., :half] + size[..., half:2 * half]
        reach = torch.cat([pair, pair, size[..., 2 * half:] * 0], -1)
    else:
        pair = size[..., 0:2 * half:2] + size[..., 1:2 * half:2]
        reach = torch.cat([torch.stack([pair, pair], -1).flatten(-2), size[..., 2 * half:] * 0], -1)
    off = (got.double().cpu() - want).abs()
    angle = 2.0 ** -51 * positions.abs().double()[:, None, None] * inv_freq.double().max().item()
    assert (off <= 2.0 ** -8 * want.abs() + (1e-6 + angle) * factor * reach).all(), off.max()
    assert torch.equal(got[..., 2 * half:].cpu(), x[..., 2 * half:].cpu())      # copied as they are


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("T,H,Hk,D,rot,far", [(1, 8, 2, 128, 128, 5), (3, 4, 4, 64, 16, 2 ** 20), (17, 5, 1, 80, 32, 1000),
                                              (130, 3, 3, 256, 256, 100000), (9001, 2, 1, 64, 64, 2 ** 34)])
def test_rope(device, T, H, Hk, D, rot, far, neox):
    import sgl_kernel

    g = torch.Generator().manual_seed(T)
    q, k = torch.randn(T, H, D, generator=g).bfloat16().to(DEV), torch.randn(T, Hk, D, generator=g).bfloat16().to(DEV)
    positions = torch.randint(-far, far, (T,), generator=g)
    positions[0] = 0
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    for inv_freq, factor in ((f.to(DEV), 1.0), (f.float().to(DEV), 1.3)):
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        sgl_kernel.rotary_embedding_scaled(positions.to(DEV), q, k, inv_freq, factor, neox, qo, ko)
        check_rope(q, qo, positions, inv_freq, factor, neox)
        check_rope(k, ko, positions, inv_freq, factor, neox)
    qi, ki = q.clone(), k.clone()                        # in place: the same bits
    sgl_kernel.rotary_embedding_scaled(positions.to(DEV), qi, ki, inv_freq, factor, neox)
    assert torch.equal(qi, qo) and torch.equal(ki, ko)


def test_rope_on_slices_of_a_fused_projection(device):
    import sgl_kernel

    T, H, Hk, D = 33, 6, 2, 128
    qkv = torch.randn(T, (H + 2 * Hk) * D, device=DEV).bfloat16()
    keep = qkv.clone()
    q, k = qkv[:, :H * D].view(T, H, D), qkv[:, H * D:(H + Hk) * D].view(T, Hk, D)
    f = (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).to(DEV)
    positions = torch.arange(T, device=DEV) * 7
    sgl_kernel.rotary_embedding_scaled(positions, q, None, f, 1.0, True)
    assert torch.equal(qkv[:, H * D:], keep[:, H * D:])
    check_rope(keep[:, :H * D].view(T, H, D), q, positions, f, 1.0, True)
    sgl_kernel.rotary_embedding_scaled(positions[:0], q[:0], k[:0], f)          # no tokens
    # queries transposed from [H, T, D]
    qt = keep[:, :H * D].view(T, H, D).permute(1, 0, 2).contiguous().permute(1, 0, 2)
    sgl_kernel.rotary_embedding_scaled(positions, qt, k, f, 1.0, True)
    assert torch.equal(qt, q)


def test_rope_agrees_with_the_cached_form(device):
    """Small positions: the same rotation as rotary_embedding from an fp32 table of cosines, to the
    rounding of either."""
    import sgl_kernel

    T, H, D = 40, 4, 128
    q = torch.randn(T, H, D, device=DEV).bfloat16()
    f = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).to(DEV)
    positions = torch.arange(T, device=DEV)
    angle = positions.double()[:, None] * f[None]
    cache = torch.cat([angle.cos(), angle.sin()], -1).float()
    want, got = q.clone(), q.clone()
    sgl_kernel.rotary_embedding(positions, want.view(T, -1), None, D, cache, True)
    sgl_kernel.rotary_embedding_scaled(positions, got, None, f)
    off = (got.double() - want.double()).abs()
    assert (off <= 2.0 ** -7 * want.double().abs() + 2e-6 * 8).all()


# ----------------------------------------------------------------------------------- store --
def empty_cache(blocks, block, heads, dim, seed=0, order="thd"):
    """Codes and scales from earlier use; order "htd": heads outside tokens, as a view."""
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn(blocks, block, heads, dim, generator=g) * 80).clamp(-448, 448).to(FP8)
    scale = torch.exp2(torch.randint(-9, -4, (blocks, heads), generator=g).float())
    if order == "htd":
        dev = codes.permute(0, 2, 1, 3).contiguous().to(DEV).permute(0, 2, 1, 3)
    else:
        dev = codes.to(DEV)
    return dev, scale.to(DEV)


def same(codes, want):
    got = codes.cpu().float().double()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7e9), want.nan_to_num(7e9))


def check_store(k, v, kc, vc, ks, vs, slots):
    import sgl_kernel

    want = []
    for x, codes, scale in ((k, kc, ks), (v, vc, vs)):
        c, s = codes.cpu().float().double(), scale.cpu().double()
        oracle.store(x, c, s, slots)
        want.append((c, s))
    sgl_kernel.store_kv_cache_fp8(k, v, kc, vc, ks, vs, torch.tensor(slots, dtype=torch.int64, device=DEV))
    for (c, s), codes, scale in zip(want, (kc, vc), (ks, vs)):
        assert torch.equal(scale.cpu().double(), s)
        assert same(codes, c)


def slots_of(runs, block):
    """[(block, first place, tokens)] -> slots"""
    return [b * block + off + i for b, off, n in runs for i in range(n)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("block,order", [(16, "thd"), (64, "htd"), (256, "thd"), (1024, "htd")])
def test_store(device, block, order, D):
    heads = 3
    kc, ks = empty_cache(9, block, heads, D, 1, order)
    vc, vs = empty_cache(9, block, heads, D, 2, order)
    runs = [(4, 0, block), (2, 3, block - 3), (7, block - 1, 1), (0, 0, 1), (8, 1, 1), (1, 5, 9)]
    slots = slots_of(runs, block)
    T = len(slots)
    g = torch.Generator().manual_seed(block)
    size = torch.exp(1.5 * torch.randn(T, 1, 1, generator=g))
    k, v = ((torch.randn(T, heads, D, generator=g) * size).bfloat16().to(DEV) for _ in range(2))
    check_store(k, v, kc, vc, ks, vs, slots)


def test_store_token_by_token_and_with_a_block_used_again(device):
    """A block that fills over several calls, values growing and shrinking, then started anew."""
    block, heads, D = 16, 2, 64
    kc, ks = empty_cache(3, block, heads, D, 3)
    vc, vs = empty_cache(3, block, heads, D, 4)
    g = torch.Generator().manual_seed(5)
    for i, size in enumerate([1.0, 0.01, 300.0, 1e4, 1.0, 2.0 ** 100, 1.0]):
        k, v = ((torch.randn(1, heads, D, generator=g) * size).bfloat16().to(DEV) for _ in range(2))
        check_store(k, v, kc, vc, ks, vs, [block + i])
    k, v = ((torch.randn(2, heads, D, generator=g)).bfloat16().to(DEV) for _ in range(2))
    check_store(k, v, kc, vc, ks, vs, [block, block + 1])


def test_store_many_tokens(device):
    """The form for many tokens (runs longer and shorter than the groups that waves look at)."""
    block, heads, D = 32, 2, 128
    lens, table = [1000, 1, 33, 640, 17, 500, 32, 31], 0
    slots, used = [], 0
    for n in lens:
        first = 5 if n % 2 else 0
        for i in range(n):
            slots.append((used + (first + i) // block) * block + (first + i) % block)
        used += -(-(first + n) // block)
    slots[900:900] = [-1] * 40
    slots += [-1, used * block + 3, 2 ** 40, -2 ** 40] + [-1] * 20
    assert len(slots) > 2048
    kc, ks = empty_cache(used, block, heads, D, 6)
    vc, vs = empty_cache(used, block, heads, D, 7)
    k, v = (torch.randn(len(slots), heads, D).bfloat16().to(DEV) for _ in range(2))
    # the skipped tokens cut block 900 // 32 of the first request: its two runs are no longer one
    whole = [s for s in slots]
    cut = [i for i in range(len(whole)) if 0 <= whole[i] < used * block and whole[i] // block == whole[899] // block]
    for i in cut:
        if i > 900:
            whole[i] = -1
    check_store(k, v, kc, vc, ks, vs, whole)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("block,requests,longest", [(16, 5, 3), (16, 700, 2), (64, 300, 40), (128, 20, 300), (256, 900, 1),
                                                    (512, 9, 600)])
def test_store_of_many_requests(device, block, requests, longest, D):
    """Runs of one token to whole blocks side by side, most of them behind tokens of earlier calls,
    with the rotation, against the two operators apart."""
    import sgl_kernel

    heads = 2
    g = torch.Generator().manual_seed(block + requests)
    lens = torch.exp(torch.rand(requests, generator=g) * math.log(longest + 0.99)).int().tolist()
    slots, used = [], 0
    for n in lens:
        first = int(torch.randint(0, block, (1,), generator=g))
        slots += [(used + (first + i) // block) * block + (first + i) % block for i in range(n)]
        used += -(-(first + n) // block)
    T = len(slots)
    kc, ks = empty_cache(used, block, heads, D, 16)
    vc, vs = empty_cache(used, block, heads, D, 17)
    size = torch.exp(2.0 * torch.randn(T, 1, 1, generator=g))
    k, v = ((torch.randn(T, heads, D, generator=g) * size).bfloat16().to(DEV) for _ in range(2))
    f = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).to(DEV)
    positions = torch.randint(0, 100000, (T,), generator=g).to(DEV)
    both = [t.clone() for t in (kc, vc, ks, vs)]
    sgl_kernel.store_kv_cache_fp8(k, v, *both, torch.tensor(slots, device=DEV), None, positions, f)
    turned = k.clone()
    sgl_kernel.rotary_embedding_scaled(positions, turned, None, f)
    check_store(turned, v, kc, vc, ks, vs, slots)
    for a, b in zip((kc, vc, ks, vs), both):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_store_values_at_the_edges(device):
    """Zeros, the borders of a power of two, tiny and huge values, infinities and NaN."""
    block, heads, D = 16, 1, 64
    rows = [0.0, -0.0, 448.0, 450.0, 224.0, 225.0, 2.0 ** -60, 2.0 ** -133, 3.3e38, -3.3e38]
    for n, x in enumerate(rows):
        kc, ks = empty_cache(2, block, heads, D, 8)
        vc, vs = empty_cache(2, block, heads, D, 9)
        k = torch.randn(2, heads, D).bfloat16().to(DEV) * (0.0 if abs(x) < 1 else 1.0)
        k[1, 0, n] = x
        v = torch.full((2, heads, D), x).bfloat16().to(DEV)
        check_store(k, v, kc, vc, ks, vs, [16, 17])
    kc, ks = empty_cache(2, block, heads, D, 10)
    vc, vs = empty_cache(2, block, heads, D, 11)
    k, v = (torch.randn(3, heads, D).bfloat16().to(DEV) for _ in range(2))
    k[0, 0, 3], k[1, 0, 5], k[2, 0, 7] = math.inf, -math.inf, math.nan
    v[1] = math.nan
    check_store(k, v, kc, vc, ks, vs, [4, 5, 6])
    k2, v2 = (torch.full((1, heads, D), 1e5).bfloat16().to(DEV) for _ in range(2))
    check_store(k2, v2, kc, vc, ks, vs, [7])             # NaN codes stay NaN when the step grows


def test_store_from_strided_rows(device):
    heads, D, T, block = 2, 128, 21, 16
    qkv = torch.randn(T, 8 * D, device=DEV).bfloat16()
    k, v = qkv[:, 4 * D:6 * D].view(T, heads, D), qkv[:, 6 * D:].view(T, heads, D)
    kc, ks = empty_cache(4, block, heads, D, 12)
    vc, vs = empty_cache(4, block, heads, D, 13)
    check_store(k, v, kc, vc, ks, vs, slots_of([(3, 0, 16), (1, 0, 5)], block))
    check_store(k[:0], v[:0], kc, vc, ks, vs, [])        # no tokens


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("D,rot,T", [(128, 128, 5), (128, 48, 37), (64, 64, 2100), (64, 16, 3)])
def test_store_with_rotation_is_the_two_operators(device, D, rot, T, neox):
    """Bit for bit: keys rotated, then stored; queries as the rotary operator gives them."""
    import sgl_kernel

    H, heads, block = 5, 2, 64
    blocks = -(-T // block) + 1
    f = (500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).to(DEV)
    q = torch.randn(T, H, D, device=DEV).bfloat16()
    k, v = (torch.randn(T, heads, D, device=DEV).bfloat16() for _ in range(2))
    positions = torch.arange(T, device=DEV) + 70001
    slots = torch.arange(T, device=DEV) + block
    kc, ks = empty_cache(blocks, block, heads, D, 14)
    vc, vs = empty_cache(blocks, block, heads, D, 15)
    both = [t.clone() for t in (kc, vc, ks, vs)]
    qo, keep = torch.empty_like(q), (k.clone(), v.clone())
    sgl_kernel.store_kv_cache_fp8(k, v, kc, vc, ks, vs, slots, q, positions, f, 1.1, neox, qo)
    assert torch.equal(k, keep[0]) and torch.equal(v, keep[1])
    q2, k2 = q.clone(), k.clone()
    sgl_kernel.rotary_embedding_scaled(positions, q2, k2, f, 1.1, neox)
    sgl_kernel.store_kv_cache_fp8(k2, v, both[0], both[1], both[2], both[3], slots)
    assert torch.equal(qo, q2)
    for a, b in zip((kc, vc, ks, vs), both):
        assert torch.equal(a.view(torch.uint8) if a.dtype == FP8 else a, b.view(torch.uint8) if b.dtype == FP8 else b)
    # without queries, and queries in place
    sgl_kernel.store_kv_cache_fp8(k, v, kc, vc, ks, vs, slots, None, positions, f, 1.1, neox)
    sgl_kernel.store_kv_cache_fp8(k, v, kc, vc, ks, vs, slots, q, positions, f, 1.1, neox)
    assert torch.equal(q, q2)


# ---------------------------------------------------------------------------------- attend --
class Case:
    """Sequences in a paged cache; everything behind their ends is NaN."""

    def __init__(self, new, lens, H, Hk, D, block, seed=0, order="thd", spread=0, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.new, self.lens, self.H, self.Hk, self.D, self.block = new, lens, H, Hk, D, block
        need = [-(-max(n, 0) // block) for n in lens]
        self.blocks = sum(need) + spare
        codes = [(torch.randn(self.blocks, block, Hk, D, generator=g) * 90).clamp(-448, 448) for _ in range(2)]
        scales = [torch.exp2(torch.randint(-9 - spread, -5 + spread, (self.blocks, Hk), generator=g).float())
                  for _ in range(2)]
        order_of = torch.randperm(self.blocks, generator=g).tolist()
        self.table = torch.full((len(lens), max(need + [1]) + 1), 2 ** 30, dtype=torch.int32)
        at, used = 0, set()
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(order_of[at:at + n], dtype=torch.int32)
            used |= set(order_of[at:at + n])
            at += n
            if lens[b] > 0 and lens[b] % block:
                for c in codes:
                    c[order_of[at - 1], lens[b] % block:] = math.nan
        for free in set(range(self.blocks)) - used:
            for c, s in zip(codes, scales):
                c[free], s[free] = math.nan, math.nan
        self.codes = [c.to(FP8) for c in codes]
        self.scales = scales
        self.cu = [sum(new[:i]) for i in range(len(new) + 1)]
        self.q = torch.randn(self.cu[-1], H, D, generator=g).bfloat16()
        if order == "htd":
            self.dev = [c.permute(0, 2, 1, 3).contiguous().to(DEV).permute(0, 2, 1, 3) for c in self.codes]
        else:
            self.dev = [c.to(DEV) for c in self.codes]

    def call(self, causal=True, window=-1, q=None, out=None, **more):
        import sgl_kernel

        q = self.q.to(DEV) if q is None else q
        args = dict(cache_seqlens=i32(self.lens), page_table=self.table.to(DEV), k_descale=self.scales[0].to(DEV),
                    v_descale=self.scales[1].to(DEV), causal=causal,
                    window_size=(window, -1 if window < 0 else 0), return_softmax_lse=True)
        if q.dim() == 3:
            args.update(cu_seqlens_q=i32(self.cu), max_seqlen_q=max(self.new + [0]))
        args.update(more)
        got, lse, *_ = sgl_kernel.flash_attn_with_kvcache(q, *self.dev, **args)
        return got, lse

    def want(self, causal=True, window=-1, scale=None):
        return oracle.attend(self.q.to(DEV), *[c.to(DEV).float() for c in self.codes], *[s.to(DEV) for s in self.scales],
                             self.table, self.lens, self.cu, self.D ** -0.5 if scale is None else scale, causal, window)

    def compare(self, got, lse, want):
        out, want_lse, mass = (t[:self.cu[-1]] if t.dim() == 3 else t[:, :self.cu[-1]] for t in want)
        got, lse = got[:self.cu[-1]].double(), lse[:, :self.cu[-1]].double()
        assert torch.equal(torch.isnan(got), torch.isnan(out))
        v_max = max((c.float().nan_to_num(0).abs() * s.nan_to_num(0)[:, None, :, None]).max().item()
                    for c, s in zip(self.codes[1:], self.scales[1:]))
        keys = max(self.lens + [0])
        bound = 2.0 ** -8 * out.abs() + 8e-4 * mass + keys * 2.0 ** -25 * v_max
        off = (got - out).abs()
        assert ((off <= bound) | torch.isnan(out)).all(), (off - bound).nan_to_num(0).max().item()
        none = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, none)
        assert (((lse - want_lse).abs() <= 4e-4) | none | torch.isnan(want_lse)).all()

    def check(self, causal=True, window=-1, **more):
        got, lse = self.call(causal, window, **more)
        self.compare(got, lse, self.want(causal, window))
        return got, lse


RAGGED = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000, 0, 300]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk,block", [(4, 4, 16), (8, 1, 32), (6, 2, 64), (16, 1, 128), (14, 2, 256)])
def test_attend_one_token(device, H, Hk, block, D):
    Case([1] * len(RAGGED), RAGGED, H, Hk, D, block, H).check()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,H,Hk,block", [([2, 5, 1, 3], 6, 2, 16), ([4, 0, 4, 4], 8, 1, 64), ([3, 1, 2, 2], 20, 2, 32)])
def test_attend_a_few_tokens(device, new, H, Hk, block, D):
    c = Case(new, [70, 513, 4, 200], H, Hk, D, block, 3)
    c.check()
    c.check(window=20)
    c.check(causal=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,lens,H,Hk,block", [
    ([64], [64], 2, 2, 64), ([129, 1, 300], [129, 1, 300], 4, 2, 16), ([33, 77, 0, 260], [400, 77, 9, 1000], 8, 2, 32),
    ([513], [2049], 5, 1, 128), ([200, 40], [200, 41], 1, 1, 1024)])
def test_attend_prompts(device, new, lens, H, Hk, block, D):
    c = Case(new, lens, H, Hk, D, block, 5)
    c.check()
    c.check(window=37)
    c.check(window=0)
    c.check(causal=False)


@pytest.mark.parametrize("new,lens,H,Hk", [
    ([1500, 100, 0, 2000, 700, 1], [1500, 900, 5, 2100, 700, 3], 64, 32),     # longest first
    ([130] * 3 + [260] * 14, [130] * 3 + list(range(260, 1660, 100)), 64, 32),  # more than are put in order
    ([1500, 1900, 40], [1300, 1900, 0], 64, 64),                               # rows before the first key
])
def test_attend_enough_prompts_to_leave_keys_whole(device, new, lens, H, Hk):
    c = Case(new, lens, H, Hk, 64, 64, 16)
    c.check()
    c.check(window=333)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk", [(8, 1), (9, 3), (4, 4), (32, 8), (6, 6)])
def test_attend_long_cache_for_each_number_of_heads(device, H, Hk, D):
    """Heads side by side in a workgroup and waves that take turns, over keys that are split."""
    c = Case([1, 2, 1], [2500, 700, 4000], H, Hk, D, 32, 17)
    c.check()
    c.check(window=1000)


@pytest.mark.parametrize("B,new,block", [(300, 1, 16), (300, 4, 64), (130, 40, 16)])
def test_attend_many_sequences(device, B, new, block):
    """More sequences than lanes, short and long."""
    g = torch.Generator().manual_seed(B)
    lens = torch.exp(torch.rand(B, generator=g) * 6.5).int().tolist()
    lens[7], lens[-1] = 3000, 0
    Case([new] * B, lens, 4, 2, 64, block, 18).check()


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 40], [130, 7, 1]])
def test_attend_whatever_the_largest_length_is_said_to_be(device, new):
    c = Case(new, [600, 90, 333], 4, 2, 128, 16, 19)
    want = c.want()
    for said in (1, 5, 5000, None):
        c.compare(*c.call(max_seqlen_q=said), want)


@pytest.mark.parametrize("new", [[1] * 4, [30] * 4])
def test_attend_shared_blocks_and_one_length(device, new):
    """Sequences that begin with the same blocks (a prompt in common), a table of one row for all,
    and cache_seqlens as one int."""
    c = Case(new, [200] * 4, 4, 2, 64, 16, 20)
    c.table[:, :9] = c.table[0, :9]
    c.check()
    c.table = c.table[:1].expand(4, -1)
    table = c.table[:1].to(DEV).expand(4, -1)
    assert table.stride(0) == 0
    c.compare(*c.call(page_table=table, cache_seqlens=200), c.want())


def test_attend_nothing(device):
    """No sequences, no tokens, a table without columns, a pool without blocks."""
    c = Case([1, 3], [40, 70], 4, 2, 64, 16, 21)
    got, lse = c.call(q=torch.empty(0, 4, 64, dtype=torch.bfloat16, device=DEV), cu_seqlens_q=i32([0, 0, 0]))
    assert got.shape == (0, 4, 64) and lse.shape == (4, 0)
    got, lse = c.call(q=torch.empty(0, 3, 4, 64, dtype=torch.bfloat16, device=DEV), cache_seqlens=i32([]),
                      page_table=torch.empty(0, 5, dtype=torch.int32, device=DEV))
    assert got.shape == (0, 3, 4, 64) and lse.shape == (0, 4, 3)
    empty = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    got, lse = c.call(page_table=empty)
    assert (got == 0).all() and (lse == -math.inf).all()
    c.dev = [x[:0] for x in c.dev]
    got, lse = c.call(page_table=empty, k_descale=torch.empty(0, 2, device=DEV), v_descale=torch.empty(0, 2, device=DEV))
    assert (got == 0).all() and (lse == -math.inf).all()


def test_attend_into_the_memory_of_q(device):
    """`out` may be q itself: a row is read before it is written."""
    import sgl_kernel  # noqa: F401

    for new in ([1, 1], [3, 2], [100, 60]):
        c = Case(new, [3000, 400], 8, 2, 128, 32, 22)
        want, lse = c.check()
        q = c.q.to(DEV)
        got, lse2, *_ = torch.ops.sgl_kernel.fwd.default(
            q, *c.dev, None, None, None, q, i32(c.cu), None, None, None, i32(c.lens), max(new), None, c.table.to(DEV),
            None, None, None, None, None, None, c.scales[0].to(DEV), c.scales[1].to(DEV), None, True, -1, -1, 0, 0.0,
            False, None, 0, None, 0, None)
        assert got.data_ptr() == q.data_ptr() and torch.equal(q, want) and torch.equal(lse, lse2)


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [14, 9], [90, 40]])
def test_attend_bad_queries_stay_in_their_rows(device, new):
    """NaN and infinities in one row and head of q: NaN there, the others as they are."""
    c = Case(new, [700, 65], 4, 2, 128, 16, 25)
    c.q[0, 1, 5], c.q[-1, 2, 0], c.q[-1, 3, 100] = math.nan, math.inf, -math.inf
    got, lse = c.call()
    want = c.want()
    c.compare(got, lse, want)
    bad = torch.isnan(got).any(-1)
    assert bad[0, 1] and bad[-1, 2] and bad[-1, 3] and bad.sum() == 3


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30])
def test_attend_any_scale_of_the_scores(device, scale):
    for new in ([1, 1], [12, 3], [70, 9]):
        c = Case(new, [900, 70], 4, 2, 64, 32, 26)
        c.compare(*c.call(softmax_scale=scale), c.want(scale=scale))


def test_attend_no_new_tokens_in_a_padded_batch(device):
    import sgl_kernel  # noqa: F401

    c = Case([0, 0, 0], [3000, 0, 17], 4, 2, 64, 16, 27)
    for T in (5, 300):
        q = torch.full((T, 4, 64), math.nan, device=DEV).bfloat16()
        out = torch.full_like(q, 3.0)
        torch.ops.sgl_kernel.fwd.default(
            q, *c.dev, None, None, None, out, i32(c.cu), None, None, None, i32(c.lens), 1, None, c.table.to(DEV),
            None, None, None, None, None, None, c.scales[0].to(DEV), c.scales[1].to(DEV), None, True, -1, -1, 0, 0.0,
            False, None, 0, None, 0, None)
        assert (out == 3.0).all()


def test_store_into_a_pool_without_blocks(device):
    import sgl_kernel

    k = torch.randn(40, 2, 64, device=DEV).bfloat16()
    codes, scale = torch.empty(0, 16, 2, 64, device=DEV).to(FP8), torch.empty(0, 2, device=DEV)
    sgl_kernel.store_kv_cache_fp8(k, k, codes, codes.clone(), scale, scale.clone(), torch.arange(40, device=DEV))
    torch.cuda.synchronize()


def test_attend_rows_that_see_nothing(device):
    """No keys at all, and more new tokens than the cache holds: the first stand before its start."""
    for new, lens in (([1, 1, 1], [0, -4, 5]), ([6, 2], [3, 0]), ([90, 40], [70, 0])):
        c = Case(new, lens, 4, 2, 128, 16, 6)
        got, lse = c.call()
        c.lens = [max(n, 0) for n in lens]
        c.compare(got, lse, c.want())
        assert (got[lse.t() == -math.inf] == 0).all()


@pytest.mark.parametrize("new", [[1] * 5, [70, 3, 1, 140, 2]])
def test_attend_heads_outside_tokens_and_fused_queries(device, new):
    """Caches laid out [block, head, token, D], queries as slices of a fused projection."""
    c = Case(new, [300, 64, 1, 190, 77], 6, 2, 128, 32, 7, order="htd")
    T = c.cu[-1]
    wide = torch.randn(T, 10 * 128).bfloat16().to(DEV)
    wide[:, :6 * 128] = c.q.reshape(T, -1).to(DEV)
    c.check(q=wide[:, :6 * 128].view(T, 6, 128))


@pytest.mark.parametrize("n", [1, 3, 50])
def test_attend_batched_queries(device, n):
    """q [B, S, H, D] gives what the packed form gives, its log-sum-exp as [B, H, S]."""
    B = 4
    c = Case([n] * B, [200, 55, 64, 310], 4, 2, 64, 16, 8)
    got, lse = c.check()
    q4 = c.q.to(DEV).view(B, n, 4, 64)
    got4, lse4 = c.call(q=q4)
    assert torch.equal(got4.view(B * n, 4, 64), got) and torch.equal(lse4.permute(1, 0, 2).reshape(4, B * n), lse)
    # and from [B, H, S, D] storage
    got5, lse5 = c.call(q=q4.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3))
    assert torch.equal(got5, got4) and torch.equal(lse5, lse4)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 2, 100]])
def test_attend_leaves_rows_behind_the_last_sequence(device, new):
    import sgl_kernel  # noqa: F401

    c = Case(new, [100, 30, 130], 4, 2, 64, 16, 9)
    T = c.cu[-1]
    q = torch.randn(T + 9, 4, 64).bfloat16().to(DEV)
    q[:T] = c.q.to(DEV)
    q[T:] = math.nan
    out = torch.full_like(q, 5.0)
    got, lse, *_ = torch.ops.sgl_kernel.fwd.default(
        q, *c.dev, None, None, None, out, i32(c.cu), None, None, None, i32(c.lens), max(new), None, c.table.to(DEV),
        None, None, None, None, None, None, c.scales[0].to(DEV), c.scales[1].to(DEV), None, True, -1, -1, 0, 0.0,
        False, None, 0, None, 0, None)
    assert got.data_ptr() == out.data_ptr() and (out[T:] == 5.0).all()
    c.compare(out, lse, c.want())


@pytest.mark.parametrize("new", [[1, 1], [6, 2], [80, 150]])
def test_attend_long_cache_is_split_and_joined(device, new):
    """Few rows over thousands of keys, one sequence far longer than the other."""
    Case(new, [9001, 150], 8, 2, 128, 64, 10).check()
    Case(new, [9001, 150], 8, 2, 64, 16, 11).check(window=5000)


@pytest.mark.parametrize("new", [[1, 3], [9, 4], [70, 64]])
def test_attend_nan_reaches_only_rows_that_see_it(device, new):
    c = Case(new, [200, 130], 4, 1, 128, 16, 12)
    n = new[0]
    # a value of the last token, and one channel of a value some tokens before; a key of the second sequence
    def at(b, key):
        return int(c.table[b, key // c.block]), key % c.block

    c.codes[1] = c.codes[1].float()
    blk, off = at(0, 199)
    c.codes[1][blk, off] = math.nan
    blk, off = at(0, 200 - n)
    c.codes[1][blk, off, 0, 77] = math.nan
    c.codes[1] = c.codes[1].to(FP8)
    c.codes[0] = c.codes[0].float()
    blk, off = at(1, 129)
    c.codes[0][blk, off] = math.nan
    c.codes[0] = c.codes[0].to(FP8)
    c.dev = [x.to(DEV) for x in c.codes]
    got, lse = c.call()
    want = c.want()
    # a NaN key makes the whole row NaN, weights and all
    c.compare(got, lse, want)
    last = c.cu[1] - 1
    assert torch.isnan(got[last]).all()
    if n > 1:
        assert torch.isnan(got[0, :, 77]).all() and torch.isfinite(got[0, :, :77]).all()
    assert torch.isnan(got[c.cu[2] - 1]).all() and torch.isfinite(got[c.cu[1]:c.cu[2] - 1]).all()


@pytest.mark.parametrize("new", [[1, 1], [50, 40]])
def test_attend_skips_blocks_outside_the_pool(device, new):
    c = Case(new, [150, 80], 4, 2, 128, 16, 13)
    c.table[0, 3], c.table[0, 7], c.table[1, 0] = -1, c.blocks, 2 ** 31 - 1
    c.check()
    c.lens = [10 ** 9, 80]                               # longer than the table: its length counts
    c.table[0, -1] = -1
    c.table[1, -1] = -1
    got, lse = c.call()
    c.lens = [c.table.shape[1] * 16, 80]
    want = oracle.attend(c.q.to(DEV), *[x.to(DEV).float() for x in c.codes], *[s.to(DEV) for s in c.scales], c.table,
                         c.lens, c.cu, c.D ** -0.5, True, -1)
    ok = ~torch.isnan(want[0])                           # the tail of the old last block is NaN
    assert torch.equal(torch.isnan(got), ~ok)


@pytest.mark.parametrize("new", [[1, 1], [3, 5], [60, 9]])
def test_attend_scales_far_apart(device, new):
    """Value blocks that differ by 2^20, keys by 2^6, a scale of zero."""
    c = Case(new, [500, 333], 4, 2, 128, 16, 14)
    g = torch.Generator().manual_seed(1)
    c.scales[1] = torch.exp2(torch.randint(-16, 5, c.scales[1].shape, generator=g).float())
    c.scales[0] = torch.exp2(torch.randint(-13, -6, c.scales[0].shape, generator=g).float()) * 0.7
    c.scales[1][int(c.table[0, 2])] = 0.0
    c.scales[0][int(c.table[1, 1])] = 0.0
    c.check()


@pytest.mark.parametrize("D", [64, 128])
def test_attend_17_to_64_rows(device, D):
    """Two waves for each row, half of the keys of a tile each: rows that see nothing, or keys of one
    half only, blocks outside the pool in either, NaN in either, one length whole and one split."""
    c = Case([20, 12, 16, 5], [15, 5000, 37, 100], 12, 3, D, 16, 23)
    c.check()
    c.check(window=9)
    c.check(window=0)
    c.check(causal=False)
    c.table[1, 0], c.table[1, 3], c.table[2, 0], c.table[3, 4] = -1, 2 ** 30, -1, -1   # pieces 0 and 3 of tiles
    c.check()
    c = Case([20, 12, 16, 5], [150, 5000, 37, 100], 12, 3, D, 16, 24)
    c.codes = [x.float() for x in c.codes]
    for b, key, channel in ((0, 140, 3), (1, 4990, 17), (2, 31, 40), (2, 32, 41), (3, 99, 63)):
        c.codes[1][int(c.table[b, key // 16]), key % 16, :, channel] = math.nan
    c.codes = [x.to(FP8) for x in c.codes]
    c.dev = [x.to(DEV) for x in c.codes]
    got, lse = c.check()
    assert torch.isnan(got[c.cu[2] - 1, :, 17]).all() and not torch.isnan(got[c.cu[1], :, 17]).any()
    c.check(window=9)


def test_attend_scores_far_apart(device):
    """Scores of some hundreds: all weight on one key, and the reference moving tile after tile."""
    for new in ([1], [5], [100]):
        c = Case(new, [700], 2, 1, 64, 64, 15)
        got, lse = c.call(softmax_scale=4.0)
        out, want_lse, mass = c.want(scale=4.0)
        # a score of 4 Σ q k around 700 is off by 64 u 4 Σ|q k| < 64 * 2^-24 * 3000 = 1.2e-2 at worst
        off = (got.double() - out).abs()
        assert (off <= 2.0 ** -8 * out.abs() + 3e-2 * mass + 1e-6).all()
        assert ((lse.double() - want_lse).abs() <= 2e-2).all()


def test_attend_offsets_beyond_32_bits(device):
    """Blocks that begin more than 2^32 bytes into the pool."""
    import sgl_kernel

    block, Hk, D, H = 64, 8, 128, 8
    blocks = (5 << 30) // (block * Hk * D)
    kc = torch.zeros((blocks, block, Hk, D), dtype=torch.uint8, device=DEV).view(FP8)
    vc = torch.zeros((blocks, block, Hk, D), dtype=torch.uint8, device=DEV).view(FP8)
    ks, vs = (torch.ones(blocks, Hk, device=DEV) for _ in range(2))
    T = 100
    k, v = (torch.randn(T, Hk, D, device=DEV).bfloat16() for _ in range(2))
    places = torch.arange(T, device=DEV)
    table = i32([[blocks - 1, blocks - 7]])
    slots = table[0, places // block].long() * block + places % block
    sgl_kernel.store_kv_cache_fp8(k, v, kc, vc, ks, vs, slots)
    small = [torch.stack([c.view(torch.uint8)[blocks - 1], c.view(torch.uint8)[blocks - 7]]).view(FP8) for c in (kc, vc)]
    scales = [torch.stack([s[blocks - 1], s[blocks - 7]]) for s in (ks, vs)]
    for n in (1, 60):
        q = torch.randn(n, H, D, device=DEV).bfloat16()
        args = dict(cache_seqlens=i32([T]), cu_seqlens_q=i32([0, n]), max_seqlen_q=n, causal=True)
        far = sgl_kernel.flash_attn_with_kvcache(q, kc, vc, page_table=table, k_descale=ks, v_descale=vs, **args)
        near = sgl_kernel.flash_attn_with_kvcache(q, *small, page_table=i32([[0, 1]]), k_descale=scales[0],
                                                  v_descale=scales[1], **args)
        assert torch.equal(far, near)


# -------------------------------------------------------------------------- all of them --
class Step:
    """A model layer's use of the four operators on buffers of fixed size."""

    def __init__(self, B, H, Hk, D, block, blocks, width, room):
        self.H, self.Hk, self.D, self.block, self.blocks = H, Hk, D, block, blocks
        self.kc, self.ks = empty_cache(blocks, block, Hk, D, 20)
        self.vc, self.vs = empty_cache(blocks, block, Hk, D, 21)
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
        self.free = torch.randperm(blocks, generator=torch.Generator().manual_seed(3)).int().to(DEV)
        self.context, self.new, self.begin = i32([0] * B), i32([0] * B), i32([0])
        self.slots = torch.zeros(room, dtype=torch.int64, device=DEV)
        self.positions = torch.zeros(room, dtype=torch.int64, device=DEV)
        self.cu, self.lens, self.end, self.status = i32([0] * (B + 1)), i32([0] * B), i32([0]), i32([0] * 3)
        self.q, self.out = (torch.zeros(room, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        self.k, self.v = (torch.zeros(room, Hk, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        self.turned = torch.zeros_like(self.q)
        self.freq = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).to(DEV)

    def run(self, max_new):
        import sgl_kernel

        sgl_kernel.kv_block_plan(self.context, self.new, self.table, self.free, self.begin, self.block, self.blocks,
                                 self.slots, self.positions, self.cu, self.lens, self.end, self.status)
        sgl_kernel.store_kv_cache_fp8(self.k, self.v, self.kc, self.vc, self.ks, self.vs, self.slots, self.q,
                                      self.positions, self.freq, 1.0, True, self.turned)
        out, lse = sgl_kernel.flash_attn_with_kvcache(
            self.turned, self.kc, self.vc, cache_seqlens=self.lens, page_table=self.table, cu_seqlens_q=self.cu,
            max_seqlen_q=max_new, k_descale=self.ks, v_descale=self.vs, causal=True, return_softmax_lse=True)[:2]
        self.out.copy_(out)
        self.lse = lse
        self.context.copy_(self.lens)
        self.begin.copy_(self.end)

    def feed(self, new, g):
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        n = sum(new)
        for t in (self.q, self.k, self.v):
            t[:n] = torch.randn(n, *t.shape[1:], generator=g).bfloat16().to(DEV)

    def check(self, new):
        """The step's output against 64-bit attention over what the cache holds."""
        n = sum(new)
        assert self.status.tolist() == [0, 0, 0]
        cu = [sum(new[:i]) for i in range(len(new) + 1)]
        out, lse, mass = oracle.attend(self.turned[:n], self.kc.float(), self.vc.float(), self.ks, self.vs, self.table,
                                       self.lens.tolist(), cu, self.D ** -0.5, True, -1)
        off = (self.out[:n].double() - out).abs()
        assert (off <= 2.0 ** -8 * out.abs() + 8e-4 * mass + 1e-5).all()
        assert ((self.lse[:, :n].double() - lse).abs() <= 4e-4).all()


STEPS = [[40, 7, 100], [1, 1, 1], [1, 0, 1], [3, 2, 1], [1, 1, 1], [0, 60, 0], [1, 1, 1]]


def test_a_run_of_steps(device):
    """Prompts, then tokens one or a few at a time; the cache at the end holds what 64-bit rotation
    and rounding of every step's keys and values give."""
    g = torch.Generator().manual_seed(1)
    s = Step(3, 6, 2, 128, 16, 30, 12, 160)
    k_all, v_all = [[] for _ in range(3)], [[] for _ in range(3)]
    for new in STEPS:
        s.feed(new, g)
        s.run(max(new))
        s.check(new)
        at = 0
        for b, n in enumerate(new):
            k_all[b].append(s.k[at:at + n].double().cpu())
            v_all[b].append(s.v[at:at + n].double().cpu())
            at += n
    for b in range(3):
        k, v = torch.cat(k_all[b]), torch.cat(v_all[b])
        L = k.shape[0]
        assert L == s.lens[b].item()
        at = s.table[b, :-(-L // 16)].long()
        k = oracle.rotate(k, torch.arange(L), s.freq, 1.0, True)
        for want, codes, scale in ((k, s.kc, s.ks), (v, s.vc, s.vs)):
            step = scale[at].double().cpu().repeat_interleave(16, 0)[:L, :, None]
            got = (codes[at].float().double().cpu().reshape(-1, 2, 128)[:L]) * step
            # e4m3 rounds by 2^-4 relative, or 2^-10 steps below 2^-6; a few roundings as steps grow,
            # each by half a step of the larger one: 2^-4 + 2^-4 in all, and 2^-9 steps
            assert ((got - want).abs() <= (2.0 ** -3) * want.abs() + 2.0 ** -9 * step + 2.0 ** -8 * want.abs()).all()


def test_steps_in_a_captured_graph(device):
    """One captured step, replayed with new inputs, against the eager run; the second graph's
    workspace and eager work between the replays must not matter."""
    g1, g2 = torch.Generator().manual_seed(2), torch.Generator().manual_seed(2)
    eager, graph = (Step(3, 8, 2, 64, 16, 64, 20, 12) for _ in range(2))
    other = Step(2, 4, 4, 64, 16, 64, 20, 8)
    for s, g in ((eager, g1), (graph, g2)):
        s.feed([4, 3, 2], g)
        s.run(4)
    other.feed([4, 4], g1)
    other.run(4)
    g2 = torch.Generator().manual_seed(9)
    g1 = torch.Generator().manual_seed(9)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        keep = [t.clone() for t in (graph.context, graph.begin, graph.table, graph.kc.view(torch.uint8),
                                    graph.vc.view(torch.uint8), graph.ks, graph.vs)]
    torch.cuda.current_stream().wait_stream(stream)
    cg, cg2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(cg):
        graph.run(4)
    with torch.cuda.graph(cg2):
        other.run(4)
    for t, k in zip((graph.context, graph.begin, graph.table, graph.kc.view(torch.uint8), graph.vc.view(torch.uint8),
                     graph.ks, graph.vs), keep):
        t.copy_(k)
    for new in ([1, 1, 1], [4, 1, 2], [0, 0, 1], [1, 1, 1], [4, 4, 4]):
        eager.feed(new, g1)
        graph.feed(new, g2)
        eager.run(max(new))
        cg.replay()
        cg2.replay()
        torch.cuda.synchronize()
        n = sum(new)
        graph.check(new)
        for name in ("table", "slots", "positions", "cu", "lens", "end", "status", "ks", "vs"):
            assert torch.equal(getattr(eager, name), getattr(graph, name)), name
        assert torch.equal(eager.turned[:n], graph.turned[:n])
        assert torch.equal(eager.kc.view(torch.uint8), graph.kc.view(torch.uint8))


def test_two_streams(device):
    """Calls on two streams at a time, each with its own workspace."""
    cases = [Case([1] * 6, [3000, 10, 700, 64, 1, 2000], 8, 2, 128, 32, s) for s in (31, 32)]
    want = [c.check() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    devs = [c.q.to(DEV) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                got[i].append(c.call(q=devs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])
