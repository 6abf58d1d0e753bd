"""A bound for the attention over the paged 8-bit cache that a lost tile of values does not pass, also in a
long cache, where one tile is little beside Σ p |v|.

Each weight p has an error of its own: half rounds it by up to 2^-11 of it, its score in fp32 by less than
2e-4 (128 u Σ|q k| scale, u = 2^-24, for the sizes of these tests), so by r = 7e-4 of it at most.  The n
errors of a row are rounded off one by one: for independent ones within ±r p v Hoeffding's inequality leaves
  P(|Σ error| > t) <= 2 exp(-t^2 / (2 r^2 Σ p^2 v^2)),
below 1e-12 at t = 7.6 r sqrt(Σ p^2 v^2), for each of fewer than 1e6 outputs.  What errors share (the
reference, the row sum) divides out but for 2^-20 of the output.  Beside that the output's own rounding,
2^-8 of it, and what half cannot hold: a weight is off by 2^-25 at most where the row's largest is at least 2^8 (all times
value scale), which is 2^-33 448 max(value scale) for each key."""
import math

import torch

TILE = 64


def attend(case, values=None, causal=True, window=-1, device="cpu"):
    """out, log-sum-exp and bound of a Case, float64; `values` instead of the dequantised ones [blocks, block, heads, D]."""
    c = case
    T, H, D = c.q.shape
    keys_all = c.codes[0].double() * c.scales[0].double()[:, None, :, None]
    vals_all = c.codes[1].double() * c.scales[1].double()[:, None, :, None] if values is None else values
    out = torch.zeros(T, H, D, dtype=torch.float64, device=device)
    lse = torch.full((H, T), -math.inf, dtype=torch.float64, device=device)
    bound = out.clone()
    top_scale = c.scales[1].nan_to_num(0).max().item()
    for b, length in enumerate(c.lens):
        n = c.new[b]
        length = min(max(length, 0), c.table.shape[1] * c.block)
        if n == 0 or length == 0:
            continue
        rows = slice(c.cu[b], c.cu[b + 1])
        pages = c.table[b, :-(-length // c.block)].long()
        good = (pages >= 0) & (pages < c.blocks)
        live = good.repeat_interleave(c.block)[:length].to(device)
        pages = torch.where(good, pages, 0)
        key = torch.arange(length, device=device)
        place = torch.arange(length - n, length, device=device)[:, None]
        seen = live[None] & (key[None] <= place if causal else key[None] >= 0)
        if window >= 0:
            seen = seen & (key[None] >= place - window)
        for head in range(H):
            kv = head * c.Hk // H
            k = keys_all[pages, :, kv].reshape(-1, D)[:length].to(device)
            v = vals_all[pages, :, kv].reshape(-1, D)[:length].to(device)
            k, v = (torch.where(live[:, None], x, 0.0) for x in (k, v))
            s = c.q[rows, head].double().to(device) @ k.t() * D ** -0.5
            s = s.masked_fill(~seen, -math.inf)
            lse[head, rows] = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[head, rows][:, None]).nan_to_num(0)
            out[rows, head] = p @ v
            bound[rows, head] = 7.6 * 7e-4 * ((p * p) @ (v * v)).sqrt() + length * 2.0 ** -33 * 448 * top_scale
    return out, lse, bound + (2.0 ** -8 + 2.0 ** -20) * out.abs()


# new tokens, lengths, heads, key heads, head size, block, window: few rows, 17 to 64, many; split and joined
LONG = [
    ([1, 1], [9001, 1500], 8, 2, 128, 64, -1),
    ([1, 1], [9001, 1500], 8, 2, 64, 16, 5000),
    ([1], [60000], 4, 1, 128, 32, -1),
    ([6, 2], [9001, 1500], 8, 2, 128, 64, -1),
    ([6, 2], [9001, 1500], 8, 2, 64, 16, 5000),
    ([80, 150], [9001, 1500], 4, 2, 128, 64, -1),
    ([80, 150], [5001, 1500], 4, 2, 64, 16, 3000),
]


def finite(case):
    """Everything behind the sequences' ends finite too."""
    g = torch.Generator().manual_seed(77)
    for i in range(2):
        x = case.codes[i].float()
        case.codes[i] = torch.where(torch.isnan(x), torch.randn(x.shape, generator=g) * 90, x).clamp(-448, 448).to(torch.float8_e4m3fn)
        case.scales[i] = case.scales[i].nan_to_num(2.0 ** -7)
    return case


def lost_tiles(case, window=-1):
    """The first, the last and one tile between of the longest sequence that all its rows see: (key, values without it)."""
    c, b = case, case.lens.index(max(case.lens))
    first = max(0, c.lens[b] - 1 - window) if window >= 0 else 0
    last = c.lens[b] - c.new[b]
    tiles = range(-(-first // TILE), last // TILE)
    whole = c.codes[1].double() * c.scales[1].double()[:, None, :, None]
    for t in (tiles[0], tiles[len(tiles) // 2], tiles[-1]):
        v = whole.clone()
        for key in range(t * TILE, (t + 1) * TILE):
            v[int(c.table[b, key // c.block]), key % c.block] = 0.0
        yield b, t * TILE, v
