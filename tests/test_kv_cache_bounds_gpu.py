"""Attention over long caches against the 64-bit form, with the bound of kv_cache_bounds.py (its derivation is
there): every tile of values counts."""
import pytest
import torch

from tests import kv_cache_bounds as bounds
from tests.test_kv_cache_gpu import DEV, Case

pytestmark = pytest.mark.gpu


def check(c, got, lse, **how):
    out, want_lse, bound = bounds.attend(c, device=DEV, **how)
    off = (got.double() - out).abs()
    assert (off <= bound).all(), (off / bound).max().item()
    none = want_lse == -float("inf")
    assert torch.equal(lse == -float("inf"), none)
    assert (((lse.double() - want_lse).abs() <= 4e-4) | none).all()


@pytest.mark.parametrize("new,lens,H,Hk,D,block,window", bounds.LONG)
def test_long_caches(device, new, lens, H, Hk, D, block, window):
    c = bounds.finite(Case(new, lens, H, Hk, D, block, 90))
    c.dev = [x.to(DEV) for x in c.codes]
    check(c, *c.call(window=window), window=window)


@pytest.mark.parametrize("new", [[1, 1], [5, 4], [50, 40]])
def test_lengths_beyond_the_table(device, new):
    """A length that the table has no room for counts as the table's, and what its last block holds is seen."""
    c = bounds.finite(Case(new, [150, 80], 4, 2, 128, 16, 92))
    c.dev = [x.to(DEV) for x in c.codes]
    c.table[0, -1], c.table[1, -1] = int(c.table[1, 0]), -1
    c.table[0, 3] = -1
    c.lens = [10 ** 9, 2 ** 31 - 1]
    got, lse = c.call()
    check(c, got, lse)
    shorter = [c.table.shape[1] * 16] * 2
    same, lse2 = c.call(cache_seqlens=torch.tensor(shorter, dtype=torch.int32, device=DEV))
    assert torch.equal(got, same) and torch.equal(lse, lse2)
    c.lens = [shorter[0] - 1, shorter[1] - 1]
    other, _ = c.call()
    assert not torch.equal(got, other)                    # the last place is one that a row sees
