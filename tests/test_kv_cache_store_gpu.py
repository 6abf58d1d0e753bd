"""The quantising store where the tokens of a block do not follow each other in the call: skipped tokens
between them, sequences in turn, any order.  Codes and scales are exact (one rounding of an exact product
with a power of two), so there is no tolerance."""
import math

import pytest
import torch

from tests import kv_cache_oracle as oracle
from tests.test_kv_cache_gpu import DEV, empty_cache, same

pytestmark = pytest.mark.gpu


def store_blocks(x, codes, scale, slots):
    """The definition: all tokens of a call that go to a block, whatever their order, make its scale."""
    blocks, size = codes.shape[:2]
    ours = {}
    for t, s in enumerate(slots):
        if 0 <= s < blocks * size:
            ours.setdefault(s // size, []).append(t)
    x = x.double().cpu()
    for block, tokens in ours.items():
        oracle.store(x[sorted(tokens, key=lambda t: slots[t])], codes, scale, sorted(slots[t] for t in tokens))


def check(k, v, caches, slots):
    import sgl_kernel

    kc, vc, ks, vs = caches
    want = []
    for x, codes, scale in ((k, kc, ks), (v, vc, vs)):
        c, s = codes.cpu().float().double(), scale.cpu().double()
        store_blocks(x, c, s, slots)
        want.append((c, s))
    sgl_kernel.store_kv_cache_fp8(k, v, kc, vc, ks, vs, torch.tensor(slots, dtype=torch.int64, device=DEV))
    for (c, s), codes, scale in zip(want, (kc, vc), (ks, vs)):
        assert torch.equal(scale.cpu().double(), s)
        assert same(codes, c)


def caches_of(blocks, block, heads, D, seed):
    kc, ks = empty_cache(blocks, block, heads, D, seed)
    vc, vs = empty_cache(blocks, block, heads, D, seed + 1)
    return kc, vc, ks, vs


def rows(T, heads, D, seed):
    """Tokens of very different size, so that the scales of a block's pieces differ."""
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(2.0 * torch.randn(T, 1, 1, generator=g))
    return [(torch.randn(T, heads, D, generator=g) * size).bfloat16().to(DEV) for _ in range(2)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("block", [16, 64, 256, 1024])
def test_skipped_tokens_in_the_middle_of_a_block(device, block, D):
    """Rejected drafts: slots of -1 between tokens that go on at the next place, or leave one out."""
    heads = 2
    slots = []
    for b in range(4):
        place = (5 * b) % block
        while place < block:
            slots.append(b * block + place)
            if len(slots) % 3 == 0:
                slots.append(-1)
            place += 2 if len(slots) % 7 == 0 else 1
    check(*rows(len(slots), heads, D, block), caches_of(5, block, heads, D, 50), slots)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("block,sequences,tokens", [(16, 3, 5), (32, 70, 9), (128, 9, 100), (1024, 3, 900)])
def test_sequences_in_turn(device, block, sequences, tokens, D):
    """The first token of each sequence, then the second of each, behind tokens of earlier calls."""
    heads = 3
    per = -(-(tokens + 7) // block)
    slots = [(b * per) * block + b % 8 + i for i in range(tokens) for b in range(sequences)]
    check(*rows(len(slots), heads, D, tokens), caches_of(per * sequences, block, heads, D, 52), slots)


@pytest.mark.parametrize("block,blocks,T", [(16, 5, 60), (16, 900, 3000), (64, 40, 2000), (512, 11, 5000), (1024, 3, 2500)])
def test_any_order(device, block, blocks, T):
    """A random order, with slots outside the pool among them, and blocks whose numbers share their
    low bits."""
    heads, D = 2, 64
    g = torch.Generator().manual_seed(T)
    pool = blocks if blocks != 5 else 2048 * 4 + 1
    of = (lambda b: b) if blocks != 5 else (lambda b: 2048 * b)
    places = torch.randperm(blocks * block, generator=g)[:T].tolist()
    slots = [of(s // block) * block + s % block for s in places]
    for i in range(0, len(slots), 11):
        slots[i] = (-1, pool * block + 3, -2 ** 40, 2 ** 40)[i % 4]
    check(*rows(len(slots), heads, D, T), caches_of(pool, block, heads, D, 54), slots)


def test_a_block_at_both_ends_of_a_long_call(device):
    """Whole blocks in order, and one whose first token comes first and whose others come last."""
    block, heads, D = 32, 2, 128
    slots = [0] + list(range(block, 150 * block)) + [3, 1, 2]
    check(*rows(len(slots), heads, D, 1), caches_of(150, block, heads, D, 56), slots)
    slots = list(range(block, 150 * block)) + [7 + i for i in range(9)]
    slots[2000:2000] = [5, -1, 6]
    check(*rows(len(slots), heads, D, 2), caches_of(150, block, heads, D, 58), slots)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("D,rot,block", [(128, 128, 16), (128, 48, 512), (64, 64, 256)])
def test_any_order_with_rotation(device, D, rot, block, neox):
    """Bit for bit what the two operators give apart."""
    import sgl_kernel

    H, heads, T = 3, 2, 700
    blocks = -(-T // block) + 1
    g = torch.Generator().manual_seed(rot)
    f = (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).to(DEV)
    positions = torch.randint(0, 100000, (T,), generator=g).to(DEV)
    slots = torch.randperm(blocks * block, generator=g)[:T].tolist()
    slots[100:130] = [-1] * 30
    k, v = rows(T, heads, D, rot + 1)
    q = torch.randn(T, H, D, device=DEV).bfloat16()
    caches = caches_of(blocks, block, heads, D, 60)
    both = [t.clone() for t in caches]
    out = torch.empty_like(q)
    sgl_kernel.store_kv_cache_fp8(k, v, *both, torch.tensor(slots, device=DEV), q, positions, f, 1.1, neox, out)
    k2, q2 = k.clone(), q.clone()
    sgl_kernel.rotary_embedding_scaled(positions, q2, k2, f, 1.1, neox)
    check(k2, v, caches, slots)
    assert torch.equal(out, q2)
    for a, b in zip(caches, both):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_any_order_in_a_captured_graph(device):
    """Replays with other slots: nothing of an earlier order is kept."""
    import sgl_kernel

    block, heads, D, T, blocks = 16, 2, 64, 90, 9
    k, v = rows(T, heads, D, 3)
    start = caches_of(blocks, block, heads, D, 62)
    caches = [t.clone() for t in start]
    slots = torch.zeros(T, dtype=torch.int64, device=DEV)
    orders = [list(range(T))] + [torch.randperm(blocks * block, generator=torch.Generator().manual_seed(i))[:T].tolist()
                                 for i in range(3)] + [[-1] * T]
    slots.copy_(torch.tensor(orders[1]))
    sgl_kernel.store_kv_cache_fp8(k, v, *caches, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sgl_kernel.store_kv_cache_fp8(k, v, *caches, slots)
    for order in orders:
        for a, b in zip(caches, start):
            a.view(torch.uint8).copy_(b.view(torch.uint8))
        slots.copy_(torch.tensor(order))
        graph.replay()
        eager = [t.clone() for t in start]
        check(k, v, eager, order)
        for a, b in zip(caches, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_the_definition_is_that_of_the_oracle_where_tokens_are_in_order(device):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(20, 2, 64, generator=g).bfloat16()
    slots = [16 + i for i in range(9)] + [-1, -1] + [40 + i for i in range(9)]
    a, b = [(torch.zeros(4, 16, 2, 64, dtype=torch.float64), torch.ones(4, 2, dtype=torch.float64)) for _ in range(2)]
    oracle.store(x, *a, slots)
    store_blocks(x, *b, slots)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and math.isfinite(a[0].sum())
