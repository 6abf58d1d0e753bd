"""Attention over the paged 8-bit cache where single weights, scores and NaN are hard to see in the
output: against the 64-bit form (kv_cache_oracle.py), with a bound that follows each row's own weights.

The bound (u = half a step, relative: bf16 2^-8, half 2^-11, fp32 2^-24): a weight p~ is rounded to half,
relative to a reference that leaves the row's largest weight in [2^8, 2^15].  That is 2^-11 p~, and 2^-25
where p~ is subnormal.  The row sum, in fp32, is at least 2^8 / (the largest value scale), so the second
part moves an output by at most 2^-25 * 448 * 2^-8 of that scale for each key.  Scores are off by at
most 128 u Σ|q k| scale < 2e-4 for the sizes here, where nothing else is said:
  2^-8 |o| + 8e-4 Σ p |v| + keys 2^-33 448 max(value scale);  log-sum-exp 4e-4."""
import math

import pytest
import torch

from tests.test_kv_cache_gpu import Case, DEV, FP8

pytestmark = pytest.mark.gpu


def bound(c, out, mass, scores=8e-4):
    keys = max(c.lens + [0])
    top = max(s.nan_to_num(0).max().item() for s in c.scales[1:])
    return 2.0 ** -8 * out.abs() + scores * mass + keys * 2.0 ** -33 * 448 * top


def compare(c, got, lse, want):
    out, want_lse, mass = want
    got, lse = got.double(), lse.double()
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    off = (got - out).abs()
    assert ((off <= bound(c, out, mass)) | torch.isnan(out)).all(), (off - bound(c, out, mass)).nan_to_num(0).max().item()
    none = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, none) and torch.equal(torch.isnan(lse), torch.isnan(want_lse))
    assert (((lse - want_lse).abs() <= 4e-4) | none | torch.isnan(want_lse)).all()


def recode(c):
    c.codes = [x.float().to(FP8) for x in c.codes]
    c.dev = [x.to(DEV) for x in c.codes]


# ----------------------------------------------------------- one key far above all others --
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,lens,H,Hk", [
    ([1] * 300, [500] * 300, 8, 4),              # up to 16 rows, one piece
    ([1], [70000], 8, 4),                        # and split
    ([6] * 130, [400] * 130, 8, 2),              # 17 to 64 rows
    ([1500, 1700], [1500, 1700], 64, 32),        # whole prompts
])
def test_many_small_weights_behind_a_large_one(device, new, lens, H, Hk, D):
    """A first key that takes nearly all of the weight and has a value of zero, as models make them: the
    output is what the many others add up to, each some 2^-25 of the largest."""
    if len(new) == 2:
        H, Hk = (H, Hk) if D == 64 else (H // 2, Hk // 2)
    c = Case(new, lens, H, Hk, D, 64, 40)
    g = torch.Generator().manual_seed(41)
    c.codes = [torch.zeros(c.codes[0].shape), 64 + 16 * torch.randn(c.codes[1].shape, generator=g)]
    for b in range(len(lens)):
        c.codes[0][int(c.table[b, 0]), 0] = 16.0
        c.codes[1][int(c.table[b, 0]), 0] = 0.0
    c.scales = [torch.full_like(c.scales[0], 2.0 ** -4), torch.full_like(c.scales[1], 2.0 ** -6)]
    # the first key's score, 17.7 to 18.5 for each row: 25.5 to 26.7 in powers of two
    c.q = ((17.7 + 0.8 * torch.rand(c.cu[-1], H, 1, generator=g)) / D ** 0.5).expand(-1, -1, D).bfloat16()
    recode(c)
    got, lse = c.call(causal=False)
    compare(c, got, lse, c.want(causal=False))


# --------------------------------------------------------- NaN in keys that weigh nothing --
@pytest.mark.parametrize("which", ["key", "value"])
@pytest.mark.parametrize("place,large", [(100, 8500), (8500, 100)])
@pytest.mark.parametrize("new,H,Hk", [([1], 8, 2), ([5], 8, 2), ([70], 8, 2), ([70], 32, 2)])
def test_nan_far_below_the_largest_score(device, new, H, Hk, place, large, which):
    """A NaN in the cache reaches every row that sees it, also where its piece of the keys has no weight
    beside another piece: 0 * NaN is NaN, however the keys are cut."""
    c = Case(new, [9001], H, Hk, 64, 16, 42)
    c.codes = [x.float() for x in c.codes]
    c.codes[0][:] = 0.0
    c.codes[0][int(c.table[0, large // 16]), large % 16] = 16.0     # a score of 200: 2^288 times the others
    c.scales[0][:] = 2.0 ** -4
    c.q[:] = 200 / 64 ** 0.5
    at = int(c.table[0, place // 16]), place % 16
    if which == "key":
        c.codes[0][at[0], at[1], 0, 5] = math.nan
    else:
        c.codes[1][at[0], at[1], 0, 5] = math.nan
    recode(c)
    got, lse = c.call()
    first = slice(0, H // Hk)                                     # heads of the key head that has it
    if which == "key":
        assert torch.isnan(got[:, first]).all() and torch.isnan(lse[first]).all()
    else:
        assert torch.isnan(got[:, first, 5]).all() and not torch.isnan(got[:, first, :5]).any()
        assert not torch.isnan(lse).any()
    assert not torch.isnan(got[:, H // Hk:]).any()


# -------------------------------------------------------------- scores far below all else --
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,lens", [([1, 1], [3000, 70]), ([6, 2], [3000, 70]), ([90, 30], [3000, 70])])
def test_scores_far_below_any_reference(device, new, lens, D):
    """Every score below -10^33, one key the least so: a row that sees keys has their weight, however low."""
    c = Case(new, lens, 4, 2, D, 64, 43)
    c.codes = [torch.full(c.codes[0].shape, -32.0), c.codes[1].float()]
    c.scales[0][:] = 2.0 ** 50
    c.scales[1][:] = 2.0 ** -6
    c.q[:] = 1e17
    for b, key in ((0, 1234), (1, 30)):
        c.codes[0][int(c.table[b, key // 64]), key % 64] = -16.0
    c.codes[1] = c.codes[1].nan_to_num(0)
    recode(c)
    got, lse = c.call()
    out, want_lse, mass = c.want()
    assert torch.isfinite(want_lse).all() and (want_lse < -1e33).all()
    # rows that do not see the least low key have equal scores, and rounding decides between them
    rows = [t for t in range(c.cu[-1]) if not (t >= c.cu[1] and lens[1] - new[1] + t - c.cu[1] < 30)]
    off = (got.double() - out).abs()[rows]
    assert (off <= bound(c, out, mass)[rows]).all(), off.max()
    assert ((lse.double() - want_lse).abs() <= 1e-4 * want_lse.abs()).all()
