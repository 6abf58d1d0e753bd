"""The bound of kv_cache_bounds.py sees what a kernel could lose: without one tile of values, anywhere in the
cache, rows of the sequence lie outside it for every head, and nearly all do (a row whose scores happen to
leave that tile next to no weight cannot miss it)."""
import pytest
import torch

from tests import kv_cache_bounds as bounds
from tests import kv_cache_oracle as oracle
from tests import test_kv_cache_gpu as gpu


@pytest.mark.parametrize("new,lens,H,Hk,D,block,window", bounds.LONG)
def test_a_lost_tile_of_values_is_seen(monkeypatch, new, lens, H, Hk, D, block, window):
    monkeypatch.setattr(gpu, "DEV", "cpu")
    c = bounds.finite(gpu.Case(new, lens, H, Hk, D, block, 90))
    out, _, bound = bounds.attend(c, window=window)
    for b, key, values in bounds.lost_tiles(c, window):
        without, _, _ = bounds.attend(c, values, window=window)
        rows = slice(c.cu[b], c.cu[b + 1])
        outside = ((without - out).abs() > bound)[rows]
        assert outside.any(-1).any(0).all() and outside.any(-1).double().mean() > 0.95, key
        assert not ((without - out).abs() > bound)[[t for t in range(c.cu[-1]) if not rows.start <= t < rows.stop]].any()


def test_the_definition_is_that_of_the_oracle(monkeypatch):
    monkeypatch.setattr(gpu, "DEV", "cpu")
    c = bounds.finite(gpu.Case([3, 40, 1], [70, 90, 300], 4, 2, 64, 16, 91))
    c.table[1, 2], c.table[2, 3] = -1, c.blocks
    for causal, window in ((True, -1), (True, 9), (False, -1)):
        out, lse, _ = bounds.attend(c, causal=causal, window=window)
        want, want_lse, _ = oracle.attend(c.q, *[x.float() for x in c.codes], *c.scales, c.table, c.lens, c.cu, 64 ** -0.5,
                                          causal, window)
        assert torch.allclose(out, want, atol=1e-12) and torch.allclose(lse, want_lse, atol=1e-12)
