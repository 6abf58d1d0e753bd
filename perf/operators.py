"""What is measured of the operators around an 8-bit paged key/value cache.

Four operators, in the order in which one model step uses them:

  plan    block tables and slot maps built from request lengths (`sgl_kernel.kv_block_plan`)
  rope    rotary positions from scaled frequencies, both pair layouts, all or part of a head
          (`sgl_kernel.rotary_embedding_scaled`)
  store   keys rotated, keys and values rounded to e4m3 with one power-of-two scale for each
          block of tokens and head, written into the cache (`sgl_kernel.store_kv_cache_fp8`)
  attend  attention of new tokens over such a cache (`sgl_kernel.flash_attn_with_kvcache`)

With `own` false, `run` computes the plain form: elementary torch operations, fp32 (angles in
fp64), one rounding at the end.  With `own` true it makes the calls of a user of the package.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
FP8 = torch.float8_e4m3fn
SCALE_EXP_MIN = -64     # the exponent of a block without a nonzero value


# ------------------------------------------------------------------------------ the cases --
def listed():
    return [
        # the next token of one conversation: two thousand tokens of cache, latency counts
        attend("attend 1 x 1 token, 2k", 1, 32, 8, 128, 16, (1, 1), (2010, 2010), 1),
        # the next token of four long documents: few rows, a long axis to split
        attend("attend 4 x 1 token, 128k", 4, 32, 8, 128, 64, (1, 1), (90000, 131071), 2),
        # a serving batch, one token each, lengths from a first token to 16k
        attend("attend 32 x 1 token, ragged", 32, 32, 8, 128, 32, (1, 1), (0, 16383), 3),
        # drafted tokens being checked, a few for each request, with a sliding window
        attend("attend 16 x 2..6 tokens, window", 16, 64, 8, 128, 16, (2, 6), (300, 8000), 4,
               window=4095),
        # three prompts read from the start
        attend("attend 3 prompts", 3, 32, 8, 128, 64, (700, 4096), (0, 0), 5),
        # one piece of a long prompt behind what is cached already, heads of 64
        attend("attend 509 tokens behind 30k", 1, 16, 2, 64, 128, (509, 509), (30001, 30001), 6),
        # the plan of a decoding step, and that of a step that reads many prompts
        plan("plan 48 x 1 token", 48, 16, (1, 1), (1, 8000), 7),
        plan("plan 500 prompts", 500, 32, (1, 2048), (0, 300), 8),
        # one decoding step's queries and keys, and those of a long prompt far out
        rope("rope 16 tokens", 16, 32, 8, 128, 128, True, 40000),
        rope("rope 8191 tokens, part of the head", 8191, 32, 8, 128, 64, False, 1000000),
        # one decoding step's keys and values, and those of prompts
        store("store 48 x 1 token", 48, 32, 8, 128, 16, 128, True, (1, 1), (0, 8000), 9),
        store("store 12 prompts", 12, 32, 8, 128, 64, 128, True, (100, 1500), (0, 200), 10),
    ]


def attend(name, seqs, heads, kv_heads, dim, block, new, context, lens_seed, window=-1):
    return dict(name=name, op="attend", seqs=seqs, heads=heads, kv_heads=kv_heads, dim=dim, block=block,
                new_lo=new[0], new_hi=new[1], ctx_lo=context[0], ctx_hi=context[1],
                lens_seed=lens_seed, window=window)


def plan(name, seqs, block, new, context, lens_seed):
    return dict(name=name, op="plan", seqs=seqs, block=block, new_lo=new[0], new_hi=new[1],
                ctx_lo=context[0], ctx_hi=context[1], lens_seed=lens_seed)


def rope(name, tokens, heads, kv_heads, dim, rot, neox, far):
    return dict(name=name, op="rope", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot,
                neox=neox, far=far)


def store(name, seqs, heads, kv_heads, dim, block, rot, neox, new, context, lens_seed):
    return dict(name=name, op="store", seqs=seqs, heads=heads, kv_heads=kv_heads, dim=dim, block=block,
                rot=rot, neox=neox, new_lo=new[0], new_hi=new[1], ctx_lo=context[0], ctx_hi=context[1],
                lens_seed=lens_seed)


def draw(rng):
    """One more case: the same operators with heads, head sizes, block sizes and lengths spread
    over the ranges that the listed ones stand for."""
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    kv_heads = rng.choice((1, 2, 4, 8, 16))
    heads = kv_heads * rng.choice((1, 2, 4, 7, 8))
    dim = rng.choice((64, 128))
    block = rng.choice((16, 32, 64, 128, 256))
    seed = rng.randrange(1 << 30)
    op = rng.choice(("attend", "attend", "plan", "rope", "store"))
    if op == "rope":
        rot = rng.choice([r for r in (16, 32, 64, 96, 128) if r <= dim])
        tokens = spread(1, 8191 * 40 // max(40, heads + kv_heads))
        case = rope("", tokens, heads, kv_heads, dim, rot, rng.random() < 0.5, spread(tokens, 1 << 20))
    elif op == "plan":
        seqs, new = spread(1, 500), spread(1, 2048)
        case = plan("", seqs, block, (rng.choice((0, 1)), new), (rng.choice((0, 1)), spread(1, 8000)), seed)
    elif op == "store":
        new = spread(1, 1500)
        seqs = spread(1, min(64, max(1, 8000 // new)))
        case = store("", seqs, heads, kv_heads, dim, block, rng.choice((16, 32, 64, dim)),
                     rng.random() < 0.5, (1, new), (0, spread(1, 4000)), seed)
    else:
        new = 1 if rng.random() < 0.5 else spread(1, 2048)
        context = spread(1, 65536)
        seqs = spread(1, 48)
        while True:  # bounded by the largest listed cases: cache bytes, products, padded scores
            keys = seqs * (context + new)
            if (keys * kv_heads * dim <= 300e6 and 4.0 * new * keys * heads * dim <= 0.3e12
                    and new * keys * heads <= 1.2e9):
                break
            if seqs > 1:
                seqs = max(1, seqs // 2)
            elif new > 1 and rng.random() < 0.5:
                new = max(1, new // 2)
            else:
                context = max(1, context // 2)
        window = -1 if rng.random() < 0.7 else spread(16, 8192)
        case = attend("", seqs, heads, kv_heads, dim, block, (1, new), (rng.choice((0, context)), context),
                      seed, window)
    del case["name"]
    return case


def lengths(case):
    """(new tokens, tokens before them) of each request: spread over the logarithm, the first
    request with the longest of both."""
    rng = random.Random(case["lens_seed"])

    def one(lo, hi):
        return min(hi, lo + int(math.exp(rng.uniform(0, math.log(hi - lo + 1)))) - (hi > lo))

    new = [one(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    ctx = [one(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    new[0], ctx[0] = case["new_hi"], case["ctx_hi"]
    return new, ctx


def visible(n, length, window):
    """How many keys the n last of `length` tokens see, added up, and how many of the keys any
    of them sees."""
    first = length - n
    if window < 0:
        return n * first + n * (n + 1) // 2, length
    pairs = sum(min(first + i, window) + 1 for i in range(n))
    return pairs, min(length, n + window)


def work(case):
    op = case["op"]
    if op == "plan":
        new, ctx = lengths(case)
        b = case["block"]
        fresh = sum(-(-(n + c) // b) - -(-c // b) for n, c in zip(new, ctx))
        # lengths in and out, the running sum, slots and positions, the free list and the table
        return {"bytes": case["seqs"] * 16.0 + sum(new) * 16.0 + fresh * 8.0, "flops": 0.0}
    if op == "rope":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        turned = values * case["rot"] / case["dim"]
        return {"bytes": values * 4.0 + case["tokens"] * 8.0 + case["rot"] * 4.0, "flops": turned * 3.0}
    new, ctx = lengths(case)
    h, hk, d, b = case["heads"], case["kv_heads"], case["dim"], case["block"]
    if op == "store":
        t = sum(new)
        return {"bytes": t * (h * d * 4.0 + hk * d * 6.0 + 16.0) + case["rot"] * 4.0,
                "flops": t * (3.0 * (h + hk) * case["rot"] + 4.0 * hk * d)}
    pairs = keys = 0
    for n, c in zip(new, ctx):
        p, k = visible(n, n + c, case["window"])
        pairs, keys = pairs + p, keys + k
    t = sum(new)
    return {"bytes": keys * hk * d * 2.0 + keys / b * (hk * 8.0 + 4.0) + t * h * (d * 4.0 + 4.0),
            "flops": 4.0 * pairs * h * d}


# ------------------------------------------------------------------------------ the inputs --
def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def frequencies(rot, far):
    """Frequencies of a context stretched by parts: fast pairs as they were trained, slow ones
    slowed by the stretch, a ramp between; and the factor on cosine and sine that goes with it."""
    base, trained = 500000.0, 8192.0
    stretch = max(1.0, far / trained)
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    turns = trained * f / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    f = f * (keep + (1 - keep) / stretch)
    return f.to(DEV), 0.1 * math.log(stretch) + 1.0


def cache_pages(g, blocks, block, kv_heads, dim):
    """A cache as it stands in use: e4m3 values that fill their range, scales that are powers of
    two, another one for each block and head."""
    codes = torch.empty((blocks, block, kv_heads, dim), dtype=FP8, device=DEV)
    step = max(1, (1 << 27) // (block * kv_heads * dim))
    for i in range(0, blocks, step):
        n = min(step, blocks - i)
        codes[i:i + n] = (normal(g, n, block, kv_heads, dim) * 90).clamp(-448, 448).to(FP8)
    e = torch.randint(-9, -5, (blocks, kv_heads), generator=g, device=DEV)
    return codes, torch.exp2(e.float())


def scattered_table(g, case, lens, spare=3):
    """Blocks of the requests, all over the pool; -1 behind the last one of a request."""
    b = case["block"]
    need = ints([-(-n // b) for n in lens], torch.int64)
    total = int(sum(-(-n // b) for n in lens))
    width = max(1, max(-(-n // b) for n in lens))
    order = torch.randperm(total + spare, generator=g, device=DEV)[:total]
    col = torch.arange(width, device=DEV)
    held = col[None, :] < need[:, None]
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    table[held] = order.int()
    return table, total + spare


def prepare(case, seed):
    g = generator(seed)
    s = dict(case)
    if case["op"] == "rope":
        t, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        s["q"], s["k"] = normal(g, t, h, d).bfloat16(), normal(g, t, hk, d).bfloat16()
        first = torch.randint(0, max(1, case["far"] - t) + 1, (1,), generator=g, device=DEV)
        s["positions"] = first + torch.arange(t, device=DEV)
        s["inv_freq"], s["attn_factor"] = frequencies(case["rot"], case["far"])
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        return s
    new, ctx = lengths(case)
    lens = [n + c for n, c in zip(new, ctx)]
    tokens = sum(new)
    if case["op"] == "plan":
        b = case["block"]
        held = ints([-(-c // b) for c in ctx], torch.int64)
        total = sum(-(-c // b) for c in ctx)
        fresh = sum(-(-n // b) for n in lens) - total
        width = max(1, max(-(-n // b) for n in lens))
        s["num_blocks"] = total + fresh + 64
        order = torch.randperm(s["num_blocks"], generator=g, device=DEV).int()
        table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
        table[torch.arange(width, device=DEV)[None, :] < held[:, None]] = order[:total]
        s["block_table"], s["free_blocks"] = table, order[total:].contiguous()
        s["context_lens"], s["new_lens"], s["free_begin"] = ints(ctx), ints(new), ints([11])
        room = tokens + 5  # some room behind the last token, as a step of fixed size has
        s["slot_mapping"] = torch.empty(room, dtype=torch.int64, device=DEV)
        s["positions"] = torch.empty(room, dtype=torch.int64, device=DEV)
        s["cu_seqlens_q"] = torch.empty(case["seqs"] + 1, dtype=torch.int32, device=DEV)
        s["seq_lens"] = torch.empty(case["seqs"], dtype=torch.int32, device=DEV)
        s["free_end"] = torch.empty(1, dtype=torch.int32, device=DEV)
        s["status"] = torch.empty(3, dtype=torch.int32, device=DEV)
        return s
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "store":
        # only the block that a request's new tokens begin in holds earlier ones that matter
        b = case["block"]
        inside = [c % b for c in ctx]
        table, blocks = scattered_table(g, case, [i + n for i, n in zip(inside, new)])
        s["k_cache"], s["k_scale"] = cache_pages(g, blocks, b, hk, d)
        s["v_cache"], s["v_scale"] = cache_pages(g, blocks, b, hk, d)
        which = torch.repeat_interleave(torch.arange(len(new), device=DEV), ints(new, torch.int64))
        starts = ints([sum(new[:i]) for i in range(len(new))], torch.int64)
        nth = torch.arange(tokens, device=DEV) - starts[which]
        at = nth + ints(inside, torch.int64)[which]
        s["slot_mapping"] = table[which, at // b].long() * b + at % b
        s["positions"] = nth + ints(ctx, torch.int64)[which]
        size = torch.exp(0.7 * normal(g, tokens, 1, 1))  # some tokens are larger than others
        s["k"], s["v"] = ((normal(g, tokens, hk, d) * size).bfloat16() for _ in range(2))
        s["q"] = normal(g, tokens, h, d).bfloat16()
        s["q_out"] = torch.empty_like(s["q"])
        s["inv_freq"], s["attn_factor"] = frequencies(case["rot"], max(lens))
        return s
    s["page_table"], blocks = scattered_table(g, case, lens)
    s["k_cache"], s["k_scale"] = cache_pages(g, blocks, case["block"], hk, d)
    s["v_cache"], s["v_scale"] = cache_pages(g, blocks, case["block"], hk, d)
    s["q"] = normal(g, tokens, h, d).bfloat16()
    s["seq_lens"] = ints(lens)
    s["cu_seqlens_q"] = ints([sum(new[:i]) for i in range(len(new) + 1)])
    s["max_new"], s["max_len"] = max(new), max(lens)
    return s


# --------------------------------------------------------------------------------- one pass --
def run(s):
    if own:
        return OWN[s["op"]](s)
    return PLAIN[s["op"]](s)


def package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang-diffusion_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import sgl_kernel

    return sgl_kernel


def own_plan(s):
    package().kv_block_plan(s["context_lens"], s["new_lens"], s["block_table"], s["free_blocks"],
                            s["free_begin"], s["block"], s["num_blocks"], s["slot_mapping"],
                            s["positions"], s["cu_seqlens_q"], s["seq_lens"], s["free_end"], s["status"])
    return {n: s[n] for n in ("block_table", "slot_mapping", "positions", "cu_seqlens_q", "seq_lens",
                              "free_end", "status")}


def own_rope(s):
    package().rotary_embedding_scaled(s["positions"], s["q"], s["k"], s["inv_freq"], s["attn_factor"],
                                      s["neox"], s["q_out"], s["k_out"])
    return {"q": s["q_out"], "k": s["k_out"]}


def own_store(s):
    package().store_kv_cache_fp8(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                 s["slot_mapping"], s["q"], s["positions"], s["inv_freq"],
                                 s["attn_factor"], s["neox"], s["q_out"])
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"], "k_scale": s["k_scale"],
            "v_scale": s["v_scale"]}


def own_attend(s):
    out, lse, *_ = package().flash_attn_with_kvcache(
        s["q"], s["k_cache"], s["v_cache"], cache_seqlens=s["seq_lens"], page_table=s["page_table"],
        cu_seqlens_q=s["cu_seqlens_q"], max_seqlen_q=s["max_new"], k_descale=s["k_scale"],
        v_descale=s["v_scale"], softmax_scale=s["dim"] ** -0.5, causal=True,
        window_size=(s["window"], -1 if s["window"] < 0 else 0), return_softmax_lse=True)
    return {"out": out, "lse": lse}


OWN = {"plan": own_plan, "rope": own_rope, "store": own_store, "attend": own_attend}


def plain_plan(s):
    b = s["block"]
    ctx, new = s["context_lens"].long(), s["new_lens"].long()
    end = torch.cumsum(new, 0)
    total = ctx + new
    held, need = (ctx + b - 1) // b, (total + b - 1) // b
    fresh = need - held
    fresh_end = torch.cumsum(fresh, 0)
    begin = s["free_begin"].long()
    lacking = (begin + fresh_end[-1:] - s["free_blocks"].numel()).clamp(min=0)
    over = (end[-1:] - s["slot_mapping"].numel()).clamp(min=0)
    wide = (need > s["block_table"].shape[1]).sum().reshape(1)
    status = torch.cat([lacking, over, wide])
    good = (status == 0).all()
    # the table: fresh blocks of request b are the list's entries from begin + (sum before b)
    col = torch.arange(s["block_table"].shape[1], device=DEV)
    at = begin + (fresh_end - fresh)[:, None] + col[None, :] - held[:, None]
    is_fresh = (col[None, :] >= held[:, None]) & (col[None, :] < need[:, None]) & good
    picked = s["free_blocks"][at.clamp(0, s["free_blocks"].numel() - 1)]
    table = torch.where(is_fresh, picked, s["block_table"])
    # one row for each new token: the request it belongs to, its place, its slot
    t = torch.arange(s["slot_mapping"].numel(), device=DEV)
    row = torch.searchsorted(end, t, right=True)
    used = (row < ctx.numel()) & good
    row = row.clamp(max=ctx.numel() - 1)
    place = ctx[row] + t - (end - new)[row]
    entry = table[row, (place // b).clamp(0, col.numel() - 1)].long()
    used_slot = used & (entry >= 0) & (entry < s["num_blocks"])
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    return {"block_table": table, "slot_mapping": torch.where(used_slot, entry * b + place % b, -1),
            "positions": torch.where(used, place, 0),
            "cu_seqlens_q": (torch.cat([zero, end]) * good).int(),
            "seq_lens": torch.where(good, total, ctx).int(),
            "free_end": (begin + fresh_end[-1:] * good).int(), "status": status.int()}


def turned(x, positions, inv_freq, factor, neox):
    """The rotation in fp32 with angles in fp64, not rounded."""
    rot = 2 * inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq[None, :]
    c, n = (angle.cos() * factor).float()[:, None, :], (angle.sin() * factor).float()[:, None, :]
    x = x.float()
    a, z = (x[..., :rot // 2], x[..., rot // 2:rot]) if neox else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, w = a * c - z * n, z * c + a * n
    both = torch.cat([u, w], -1) if neox else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([both, x[..., rot:]], -1)


def plain_rope(s):
    args = s["positions"], s["inv_freq"], s["attn_factor"], s["neox"]
    return {"q": turned(s["q"], *args).bfloat16(), "k": turned(s["k"], *args).bfloat16()}


def plain_store(s):
    args = s["positions"], s["inv_freq"], s["attn_factor"], s["neox"]
    k_scale, v_scale = s["k_scale"], s["v_scale"]
    k_cache, k_scale = put(turned(s["k"], *args).bfloat16(), s["k_cache"], k_scale, s["slot_mapping"])
    v_cache, v_scale = put(s["v"], s["v_cache"], v_scale, s["slot_mapping"])
    return {"q": turned(s["q"], *args).bfloat16(), "k_cache": k_cache, "v_cache": v_cache,
            "k_scale": k_scale, "v_scale": v_scale}


def put(x, cache, scale, slots):
    """x [T, heads, dim] into the cache.  A block's scale is the smallest power of two with
    which its largest value stays within 448; it never shrinks while the block fills, and when
    it grows, what the block holds is rounded to the larger step."""
    blocks, size, heads, dim = cache.shape
    x = x.float()
    where, off = slots // size, slots % size
    largest = torch.zeros((blocks, heads), device=DEV)
    largest.index_reduce_(0, where, x.abs().amax(-1), "amax")
    first = torch.full((blocks,), size, dtype=torch.int64, device=DEV)
    first.index_reduce_(0, where, off, "amin")
    mantissa, e = torch.frexp(largest)
    e = torch.where(largest > 0, e - 9 + (mantissa > 0.875).int(), SCALE_EXP_MIN).clamp(min=SCALE_EXP_MIN)
    fits = torch.exp2(e.float())
    touched, fresh = (first < size)[:, None], (first == 0)[:, None]
    grown = torch.where(fresh, fits, torch.maximum(scale, fits))
    new_scale = torch.where(touched, grown, scale)
    before = torch.arange(size, device=DEV)[None, :] < first[:, None]
    again = (before & touched)[:, :, None, None]
    values = cache.float()
    kept = values * torch.where(again, (scale / new_scale)[:, None, :, None], 1.0)
    kept.view(-1, heads, dim)[slots] = x / new_scale[where][:, :, None]
    cache.copy_(kept.clamp(-448, 448).to(FP8))
    scale.copy_(new_scale)
    return cache, scale


def plain_attend(s):
    h, hk, d, b = s["heads"], s["kv_heads"], s["dim"], s["block"]
    n, length = s["max_new"], s["max_len"]
    lens, cu = s["seq_lens"].long(), s["cu_seqlens_q"].long()
    new = cu[1:] - cu[:-1]
    seqs = lens.numel()
    # keys and values of each request side by side, zeros behind the last one
    j = torch.arange(length, device=DEV)
    live = j[None, :] < lens[:, None]
    page = torch.where(live, s["page_table"].long()[:, j // b], 0)
    slot = page * b + j % b

    def values(cache, scale):
        codes = cache.view(torch.uint8).view(-1, hk, d)[slot].view(FP8).float()
        return torch.where(live[:, :, None, None], codes * scale[page][..., None], 0.0)

    keys = values(s["k_cache"], s["k_scale"]).permute(0, 2, 3, 1)        # [seqs, hk, d, length]
    i = torch.arange(n, device=DEV)
    row = (cu[:-1, None] + i[None, :]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row].view(seqs, n, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(seqs, hk, h // hk * n, d), keys) * d ** -0.5
    del keys
    score = score.view(seqs, hk, h // hk, n, length)
    place = (lens - new)[:, None] + i[None, :]
    seen = (j[None, None, :] <= place[:, :, None]) & live[:, None, :]
    if s["window"] >= 0:
        seen &= j[None, None, :] >= place[:, :, None] - s["window"]
    seen = seen[:, None, None]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = weight.sum(-1, keepdim=True)
    vals = values(s["v_cache"], s["v_scale"]).permute(0, 2, 1, 3)        # [seqs, hk, length, d]
    o = torch.matmul(weight.view(seqs, hk, h // hk * n, length), vals).view(seqs, hk, h // hk, n, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(seqs, n, h, d)
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(seqs, n, h)
    t = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    nth = t - cu[seq]
    return {"out": o[seq, nth].bfloat16(), "lse": lse[seq, nth].t().contiguous()}


PLAIN = {"plan": plain_plan, "rope": plain_rope, "store": plain_store, "attend": plain_attend}


# ------------------------------------------------------------------- the definition, 64 bits --
def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    return {"rope": exact_rope, "store": exact_store, "attend": exact_attend}[case["op"]](s)


def exact_turn(s, x):
    """Pairs as complex numbers, multiplied by factor * e^(i angle)."""
    x = x.double().clone()
    half = s["inv_freq"].numel()
    angle = torch.outer(s["positions"].double(), s["inv_freq"])
    unit = torch.polar(torch.full_like(angle, s["attn_factor"]), angle)[:, None, :]
    one, two = (slice(0, half), slice(half, 2 * half)) if s["neox"] else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    pair = torch.complex(x[..., one], x[..., two]) * unit
    x[..., one], x[..., two] = pair.real, pair.imag
    return x


def exact_rope(s):
    return {"q": exact_turn(s, s["q"]), "k": exact_turn(s, s["k"])}


def e4m3(v):
    """The nearest e4m3 value (ties to even) of doubles within +-448: steps of 2^(e-3) from
    2^e to 2^(e+1), of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exact_store(s):
    done = {"q": exact_turn(s, s["q"])}
    slots = s["slot_mapping"].tolist()
    size = s["block"]
    for name, x in (("k", exact_turn(s, s["k"]).bfloat16().double()), ("v", s["v"].double())):
        cache, scale = s[name + "_cache"].double(), s[name + "_scale"].double()
        t = 0
        while t < len(slots):
            block, off = divmod(slots[t], size)
            n = 1
            while t + n < len(slots) and slots[t + n] == slots[t] + n and off + n < size:
                n += 1
            new = x[t:t + n]                                            # [n, heads, dim]
            top = new.abs().amax((0, 2))
            e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** SCALE_EXP_MIN)))
            fit = torch.exp2(e)
            if off:
                fit = torch.maximum(fit, scale[block])
                cache[block, :off] = e4m3(cache[block, :off] * (scale[block] / fit)[None, :, None])
            cache[block, off:off + n] = e4m3(new / fit[None, :, None])
            scale[block] = fit
            t += n
        done[name + "_cache"], done[name + "_scale"] = cache, scale
    return done


def exact_attend(s):
    h, hk, d, b = s["heads"], s["kv_heads"], s["dim"], s["block"]
    out = torch.zeros((s["q"].shape[0], h, d), dtype=torch.float64, device=DEV)
    lse = torch.full((h, s["q"].shape[0]), -math.inf, dtype=torch.float64, device=DEV)
    cu, lens = s["cu_seqlens_q"].tolist(), s["seq_lens"].tolist()
    for i, length in enumerate(lens):
        n = cu[i + 1] - cu[i]
        if not n or not length:
            continue
        pages = s["page_table"][i, :-(-length // b)].long()
        k, v = ((c.view(torch.uint8)[pages].view(FP8).double() * z[pages].double()[:, None, :, None])
                .reshape(-1, hk, d)[:length]
                for c, z in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
        key = torch.arange(length, device=DEV)
        place = torch.arange(length - n, length, device=DEV)[:, None]
        hidden = key[None, :] > place
        if s["window"] >= 0:
            hidden |= key[None, :] < place - s["window"]
        for head in range(h):
            kv = head * hk // h
            score = s["q"][cu[i]:cu[i + 1], head].double() @ k[:, kv].t() / math.sqrt(d)
            score = score.masked_fill(hidden, -math.inf)
            lse[head, cu[i]:cu[i + 1]] = torch.logsumexp(score, -1)
            out[cu[i]:cu[i + 1], head] = torch.softmax(score, -1) @ v[:, kv]
    return {"out": out, "lse": lse}
