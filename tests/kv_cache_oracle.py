"""Plain 64-bit forms of the operators around the paged 8-bit KV cache, on the CPU."""
import math

import torch

FP8 = torch.float8_e4m3fn


def plan(context, new, table, free, begin, block, num_blocks, room):
    """(table, slots, positions, cu, seq_lens, free_end, status) as Python lists."""
    context, new = [max(c, 0) for c in context], [max(n, 0) for n in new]
    table = [list(r) for r in table]
    begin = max(begin, 0)
    held = [-(-c // block) for c in context]
    need = [-(-(c + n) // block) for c, n in zip(context, new)]
    fresh, tokens = sum(need) - sum(held), sum(new)
    width = len(table[0]) if table else 0
    status = [min(max(0, begin + fresh - len(free)), 2 ** 31 - 1), min(max(0, tokens - room), 2 ** 31 - 1),
              sum(n > width for n in need)]  # counts that saturate
    if any(status):
        return table, [-1] * room, [0] * room, [0] * (len(new) + 1), context, begin, status
    slots, positions, cu, at = [], [], [0], begin
    for b, (c, n) in enumerate(zip(context, new)):
        for j in range(held[b], need[b]):
            table[b][j] = free[at]
            at += 1
        for p in range(c, c + n):
            e = table[b][p // block]
            slots.append(e * block + p % block if 0 <= e < num_blocks else -1)
            positions.append(p)
        cu.append(cu[-1] + n)
    pad = room - tokens
    return (table, slots + [-1] * pad, positions + [0] * pad, cu, [c + n for c, n in zip(context, new)], at, status)


def rotate(x, positions, inv_freq, factor, neox):
    """x [T, H, D] -> float64."""
    x = x.double().cpu().clone()
    half = inv_freq.numel()
    angle = positions.cpu().double()[:, None] * inv_freq.cpu().double()[None, :]
    c, s = angle.cos()[:, None] * factor, angle.sin()[:, None] * factor
    one, two = (slice(0, half), slice(half, 2 * half)) if neox else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    a, z = x[..., one].clone(), x[..., two].clone()
    x[..., one], x[..., two] = a * c - z * s, z * c + a * s
    return x


def e4m3(v):
    """Nearest e4m3 value, ties to even, of doubles; beyond 448 clamped, not finite -> NaN."""
    ok = torch.isfinite(v)
    v = torch.where(ok, v, 0.0).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(ok, torch.round(v / step) * step, math.nan)


def store(x, codes, scale, slots):
    """x [T, heads, D] (any float) into codes [blocks, block, heads, D] and scale [blocks, heads], both
    float64, in place; runs of tokens that go to one block, in their order."""
    blocks, size = codes.shape[:2]
    x = x.double().cpu()
    t = 0
    while t < len(slots):
        if not 0 <= slots[t] < blocks * size:
            t += 1
            continue
        block, n = slots[t] // size, 1
        while t + n < len(slots) and slots[t + n] >= 0 and slots[t + n] // size == block:
            n += 1
        off = [s % size for s in slots[t:t + n]]
        new = x[t:t + n]
        top = torch.where(torch.isfinite(new), new.abs(), 0.0).amax((0, 2))
        fit = torch.exp2(torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -64))))
        first = min(off)
        if first > 0:
            old = scale[block].clone()
            fit = torch.maximum(fit, old)
            shrink = torch.where(old > 0, old / fit, 1.0)
            codes[block, :first] = e4m3(codes[block, :first] * shrink[None, :, None])
        codes[block, off] = e4m3(new / fit[None, :, None])
        scale[block] = fit
        t += n


def attend(q, k_codes, v_codes, k_scale, v_scale, table, lens, cu, scale, causal, window):
    """q [T, H, D]; returns out, lse [H, T] and sum p |v| (what a relative error of the weights is
    measured against), float64; rows outside cu are NaN."""
    q = q.double()
    T, H, D = q.shape
    blocks, size, hk, _ = k_codes.shape
    out = torch.full((T, H, D), math.nan, dtype=torch.float64, device=q.device)
    mass = out.clone()
    lse = torch.full((H, T), math.nan, dtype=torch.float64, device=q.device)
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        length = min(max(length, 0), table.shape[1] * size)
        entries = table[b, :-(-length // size)].long().to(q.device)
        good = (entries >= 0) & (entries < blocks)
        at = torch.where(good, entries, 0)
        live = good.repeat_interleave(size)[:length]
        k = (k_codes[at].double() * k_scale[at].double()[:, None, :, None]).reshape(-1, hk, D)[:length]
        v = (v_codes[at].double() * v_scale[at].double()[:, None, :, None]).reshape(-1, hk, D)[:length]
        key = torch.arange(length, device=q.device)
        place = torch.arange(length - n, length, device=q.device)[:, None]
        seen = live[None, :].expand(n, length).clone()
        if causal:
            seen &= key[None, :] <= place
        if window >= 0:
            seen &= key[None, :] >= place - window
        for h in range(H):
            kv = h * hk // H
            s = torch.where(seen, q[cu[b]:cu[b + 1], h] @ k[:, kv].t() * scale, -math.inf)
            top = s.amax(-1, keepdim=True) if length else torch.full((n, 1), -math.inf, dtype=torch.float64, device=q.device)
            p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = p.sum(-1, keepdim=True)
            lse[h, cu[b]:cu[b + 1]] = (top + total.log())[:, 0]
            w = torch.where(total == 0, 0.0, p / total)  # NaN stays NaN
            # a key that a row does not see must not reach it, NaN or not
            vals = v[:, kv]
            clean = torch.where(torch.isnan(vals), 0.0, vals)
            hit = (seen.double() @ torch.isnan(vals).double()) > 0
            out[cu[b]:cu[b + 1], h] = torch.where(hit, math.nan, w @ clean)
            mass[cu[b]:cu[b + 1], h] = w @ clean.abs()
    return out, lse, mass
