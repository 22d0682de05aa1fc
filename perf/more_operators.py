"""A paged cache held in 4 bits and what a serving step does with it on one rank, in plain form and through the package.

  update_pages         page tables, lengths and slot maps of the next step, on the GPU: sequences shrink (drafts that were rejected, sequences that
                       ended), their pages return to a stack of free ones, then sequences grow by the step's new tokens
  append_kv_fp4        new keys (rotated, optionally normed) and values of a ragged batch into the cache, rounded to 4 bits, queries beside them
  paged_attention_fp4  the new tokens' queries over that cache, causally; one new token a sequence is a decode step
  unpack_fp4           a cache's values in 16 or 32 bits

A cache is codes and scales: codes [pages, page_size, kv_heads, dim / 2] bytes of two e2m1 numbers, the even channel's in the low bits, and
scales [pages, page_size, kv_heads, dim / 32], a byte e for 32 channels: 2^(e - 127), NaN for 255.  The exponent is that of the block's largest
magnitude rounded to e2m1's two significant bits, less two; numbers round to nearest even, to 6 at most.

The lengths of a batch are part of the case (`mix` seeds them), so that the work is known; page tables and contents come
from the inputs' seed.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST_EXPONENT = {"bf16": 125, "f16": 13, "f32": 125}   # 6 * 2^this is a number of the type
LEAST_EXPONENT = -125                                  # 0.5 * 2^this is a normal number in 32 bits
MOST_FLOPS = 4.12e11   # the largest listed chunk's
MOST_BYTES = 3.39e8    # the largest listed cache's
MOST_SCORES = 1.07e9   # scores that the plain form of the attention holds at once: the largest listed chunk's


def _pages(seqs, ctx, new, page, gone=0.0, short=0.0, pad=0, mix=1, **name):
    """seqs sequences of up to `ctx` tokens that stay and up to `new` that are dropped and come anew; a share `gone` of them has ended and makes
    room for prompts of up to `new`; a share `short` of the pages that the step asks for is missing; `pad` rows behind."""
    return dict(op="update_pages", seqs=seqs, ctx=ctx, new=new, page=page, gone=gone, short=short, pad=pad, mix=mix, **name)


def _batch(op, seqs, new, ctx, heads, kv_heads, dim, page, dtype, ragged=True, heads_first=True, pad=0, mix=1, **more):
    """seqs sequences of up to `new` new tokens each behind up to `ctx` cached ones (exactly so many where not ragged), `pad` rows behind
    the last sequence as a captured step of a fixed size has them; a page holds its heads one after the other, or its slots."""
    return dict(op=op, seqs=seqs, new=new, ctx=ctx, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, ragged=ragged,
                heads_first=heads_first, pad=pad, mix=mix, **more)


def _unpack(pages, page, kv_heads, dim, dtype, heads_first=True, **name):
    return dict(op="unpack_fp4", pages=pages, page=page, kv_heads=kv_heads, dim=dim, dtype=dtype, heads_first=heads_first, **name)


def listed():
    return [
        # a decode step of 64 sequences whose drafts of up to 4 tokens were rejected and come anew: launch and latency
        _pages(64, 8192, 4, 64, name="pages_64x4"),
        # a third of 96 sequences has ended and gives way to prompts of up to 4096 tokens, small pages, a padded batch: pages and slots
        _pages(96, 4096, 4096, 16, gone=0.33, pad=100, mix=2, name="pages_96x4096"),
        # a decode step of 128 sequences on one of eight ranks: norm, rotation, rounding and append in one call
        _batch("append_kv_fp4", 128, 1, 512, 8, 1, 128, 64, "bf16", norm=True, rot=128, interleaved=False, name="append_128x1"),
        # chunks of four sequences, half of a head's channels rotated in adjacent pairs, no norm
        _batch("append_kv_fp4", 4, 2048, 512, 32, 8, 128, 16, "f16", ragged=False, norm=False, rot=64, interleaved=True, name="append_4x2048_f16"),
        # odd sizes: ragged chunks of fp32 heads of 96 channels, slots before heads, a padded batch
        _batch("append_kv_fp4", 7, 300, 900, 15, 5, 96, 24, "f32", heads_first=False, pad=11, norm=True, rot=96, interleaved=False,
               name="append_7x300_f32"),
        # a few pages of one rank's cache, to be moved: latency
        _unpack(8, 64, 1, 128, "bf16", name="unpack_8x64"),
        # a whole cache of 131072 tokens back into 16 bits
        _unpack(2048, 64, 8, 128, "bf16", name="unpack_2048x64"),
        # a decode step of 64 sequences of very different lengths: the cache's bytes
        _batch("paged_attention_fp4", 64, 1, 8192, 32, 8, 128, 64, "bf16", name="decode_64x8192"),
        # one very long sequence on one of eight ranks: one key head, one token
        _batch("paged_attention_fp4", 1, 1, 262143, 8, 1, 128, 128, "bf16", ragged=False, name="decode_1x262144"),
        # a decode step of drafts of 3 tokens, small heads and pages, slots before heads
        _batch("paged_attention_fp4", 48, 3, 6000, 16, 4, 64, 16, "f16", heads_first=False, name="drafts_48x3_f16"),
        # a chunk of 4096 tokens behind 4096 cached ones: matrix instructions
        _batch("paged_attention_fp4", 1, 4096, 4096, 32, 8, 128, 64, "bf16", ragged=False, name="chunk_4096_of_8192"),
        # a batch that mixes short chunks and long ones, small heads and small pages, padded
        _batch("paged_attention_fp4", 24, 512, 2048, 12, 4, 64, 16, "f16", pad=37, mix=3, name="mixed_24x512_f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["update_pages", "append_kv_fp4", "append_kv_fp4", "unpack_fp4", "paged_attention_fp4", "paged_attention_fp4", "paged_attention_fp4"])
        page, mix, pad = rng.choice([8, 16, 16, 24, 64, 128]), rng.randint(1, 1 << 20), rng.choice([0, 0, rng.randint(1, 64)])
        dim, kv_heads = rng.choice([32, 64, 64, 96, 128, 128, 128, 192, 256]), rng.choice([1, 2, 4, 5, 8])
        heads_first = rng.random() < 0.6
        if op == "update_pages":
            c = _pages(_log(rng, 1, 1024), _log(rng, 1, 16384), _log(rng, 1, 4096), page, rng.choice([0.0, 0.0, rng.random()]),
                       rng.choice([0.0, 0.0, rng.random()]), pad, mix)
            if c["seqs"] * c["new"] > 400000:
                continue
        elif op == "unpack_fp4":
            c = _unpack(_log(rng, 1, 8192), page, kv_heads, dim, rng.choice(["bf16", "bf16", "f16", "f32"]), heads_first)
        else:
            heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
            kind = rng.choice(["decode", "chunk", "mixed"])
            seqs = {"decode": _log(rng, 1, 256), "chunk": rng.randint(1, 3), "mixed": rng.randint(2, 32)}[kind]
            new = {"decode": rng.choice([1, 1, 2, 4]), "chunk": _log(rng, 16, 4096), "mixed": _log(rng, 2, 1024)}[kind]
            append = op == "append_kv_fp4"
            ctx = _log(rng, 1, 1024 if append else (131072 if kind == "decode" else 16384))
            ragged = rng.random() < 0.7
            if append:
                c = _batch(op, seqs, new, ctx, heads, kv_heads, dim, page, rng.choice(["bf16", "bf16", "f16", "f32"]), ragged, heads_first, pad, mix,
                           norm=rng.random() < 0.5, rot=rng.choice([0, dim, dim, dim // 2]), interleaved=rng.random() < 0.3)
            else:
                c = _batch(op, seqs, new, ctx, heads, kv_heads, dim, page, rng.choice(["bf16", "bf16", "f16"]), ragged, heads_first, pad, mix)
            # what the plain form holds of keys and values, and of scores
            if seqs * (new + ctx) * kv_heads * dim > 7e8 or heads * seqs * new * (new + ctx) > MOST_SCORES:
                continue
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return c


def _lengths(case):
    """New tokens and cached ones of each sequence; update_pages: new tokens and those that stay."""
    rng = random.Random(case["mix"])
    if case["op"] == "update_pages":
        new, keep = [], []
        for _ in range(case["seqs"]):
            new.append(rng.randint(0, case["new"]))
            keep.append(0 if rng.random() < case["gone"] else rng.randint(0, case["ctx"]))
        if case["gone"]:   # those that stay decode
            new = [a if b == 0 else 1 for a, b in zip(new, keep)]
        return new, keep
    if not case["ragged"]:
        return [case["new"]] * case["seqs"], [case["ctx"]] * case["seqs"]
    return ([rng.randint(1, case["new"]) for _ in range(case["seqs"])], [rng.randint(0, case["ctx"]) for _ in range(case["seqs"])])


class State:
    """One call's inputs and what a program keeps between calls: weights, tables, caches."""


def _cos_sin(positions, rot, dev):
    """fp32 rows of rot/2 cosines and rot/2 sines, the angles in doubles."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
    a = torch.arange(positions, device=dev, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def _cache(g, dev, pages, page, heads, dim, heads_first):
    """Codes and scales of random keys or values, as appending them gives."""
    shape = (pages, heads, page) if heads_first else (pages, page, heads)
    codes = torch.empty(*shape, dim // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(*shape, dim // 32, dtype=torch.uint8, device=dev)
    for at in range(0, pages, 1024):
        part = slice(at, at + 1024)
        x = torch.randn((*codes[part].shape[:3], dim), generator=g, device=dev)
        codes[part], scales[part] = _quantized(x, 125)
    return (codes.transpose(1, 2), scales.transpose(1, 2)) if heads_first else (codes, scales)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = State()
    s.op = case["op"]
    page = case["page"]
    if s.op == "update_pages":
        new, keep = _lengths(case)
        s.page, s.tokens = page, sum(new) + case["pad"]
        held = [-(-(a + b) // page) for a, b in zip(new, keep)]
        kept = [-(-b // page) for b in keep]
        spare = 16
        order = torch.randperm(sum(held) + spare, generator=g, device=dev).to(torch.int32)
        s.table = torch.zeros((case["seqs"], max(held + [1]) + 2), dtype=torch.int32, device=dev)
        # A pass drops what the one before it added and adds as much again.  Where pages are missing, sequences start without their new tokens, and
        # others have taken pages from the stack.
        at = 0
        for b in range(case["seqs"]):
            n = kept[b] if case["short"] else held[b]
            s.table[b, :n] = order[at:at + n]
            at += n
        s.free_pages = torch.zeros(order.numel(), dtype=torch.int32, device=dev)
        asked = sum(held) - sum(kept)
        there = int(asked * (1 - case["short"])) if case["short"] else spare
        s.free_pages[:there] = order[at:at + there]
        s.free_count = torch.tensor([there], dtype=torch.int32, device=dev)
        s.keep = torch.tensor(keep, dtype=torch.int32, device=dev)
        s.new = torch.tensor(new, dtype=torch.int32, device=dev)
        s.lens = s.keep.clone() if case["short"] else s.keep + s.new
        return s
    s.dtype = dtype = DTYPES[case["dtype"]]
    hk, d = case["kv_heads"], case["dim"]
    if s.op == "unpack_fp4":
        s.codes, s.scales = _cache(g, dev, case["pages"], page, hk, d, case["heads_first"])
        return s

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype)

    hq = case["heads"]
    s.eps, s.interleaved, s.most = 1e-6, case.get("interleaved", False), MOST_EXPONENT[case["dtype"]]
    new, ctx = _lengths(case)
    lens = [a + b for a, b in zip(new, ctx)]
    starts = [0]
    for a in new:
        starts.append(starts[-1] + a)
    s.real, s.longest_new, s.longest = starts[-1], max(new), max(lens)
    t = s.real + case["pad"]
    s.starts = torch.tensor(starts, dtype=torch.int32, device=dev)
    s.lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    # pages in no order; rows of the table end where their sequence does, the rest of a row is never read
    need = [-(-a // page) for a in lens]
    order = torch.randperm(sum(need) + 3, generator=g, device=dev).to(torch.int32)
    s.table = torch.zeros((case["seqs"], max(need)), dtype=torch.int32, device=dev)
    at = 0
    for b, m in enumerate(need):
        s.table[b, :m] = order[at:at + m]
        at += m
    s.k, s.k_scales = _cache(g, dev, sum(need) + 3, page, hk, d, case["heads_first"])
    s.v, s.v_scales = _cache(g, dev, sum(need) + 3, page, hk, d, case["heads_first"])
    if s.op == "append_kv_fp4":
        # queries, keys and values are column ranges of one projection's output
        qkv = randn(t, hq + 2 * hk, d)
        s.q, s.new_k, s.new_v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        gamma = (torch.rand((2, d), generator=g, device=dev) + 0.5).to(dtype)
        s.q_gamma, s.k_gamma = (gamma[0], gamma[1]) if case["norm"] else (None, None)
        s.cos_sin = _cos_sin(s.longest, case["rot"], dev) if case["rot"] else None
    else:
        s.q = randn(t, hq, d)
        s.scale = d ** -0.5
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------

def _quantized(x, most):
    """Codes and scales of x [..., dim] in its own precision."""
    blocks = x.unflatten(-1, (-1, 32))
    fraction, exponent = torch.frexp(blocks.abs().amax(-1))          # the largest is fraction * 2^exponent, fraction in [1/2, 1)
    exponent = (exponent - 3 + (fraction >= 0.875).int()).clamp(LEAST_EXPONENT, most)
    t = torch.ldexp(blocks.abs(), -exponent[..., None])
    # steps of 1/2 below 2, of 1 below 4, of 2 from there on, each to nearest even; code k stands for MAGNITUDES[k]
    code = torch.where(t < 2, torch.round(t * 2), torch.where(t < 4, torch.round(t) + 2, torch.round(t / 2) + 4)).clamp(max=7).to(torch.uint8)
    code = (code | (torch.signbit(blocks).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, (exponent + 127).to(torch.uint8)


def _values(codes, scales):
    """What codes and scales stand for, in 32 bits."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    x = table[torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).int()]
    factor = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    factor = torch.where(scales == 255, math.nan, factor)
    return (x.unflatten(-1, (-1, 32)) * factor[..., None]).flatten(-2)


def _normed(x, gamma, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * gamma.to(x.dtype)


def _rotated(x, rows, interleaved):
    """x [T, heads, dim], rows [T, rot] of cosines and sines."""
    half = rows.size(1) // 2
    rows = rows.to(x.dtype)
    c, s = rows[:, None, :half], rows[:, None, half:]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _plain_pages(s):
    page, width, capacity = s.page, s.table.size(1), s.free_pages.numel()
    lens = s.lens.long().clamp(min=0)
    keep = torch.minimum(s.keep.long().clamp(min=0), lens)
    new = s.new.long().clamp(min=0)
    at = torch.arange(width, device=s.table.device)[None, :]
    # pages behind what stays go back, the last one first
    had, kept = ((x + page - 1).div(page, rounding_mode="floor").clamp(max=width) for x in (lens, keep))
    back = (at >= kept[:, None]) & (at < had[:, None])
    pages, count = s.table[back], s.free_count.long()[0]
    place = count + pages.numel() - 1 - torch.arange(pages.numel(), device=pages.device)
    s.free_pages[place[place < capacity]] = pages[place < capacity]
    count = (count + pages.numel()).clamp(max=capacity)
    # sequences grow in order as far as rows and pages reach
    need = (keep + new + page - 1).div(page, rounding_mode="floor") - kept
    fits = (kept + need <= width) & (keep + new <= 0x7fffffff)
    need = torch.where(fits & (new > 0), need.clamp(min=0), 0)
    rows = torch.where(fits, new, 0)
    served = fits & ((need == 0) | (need.cumsum(0) <= count)) & (rows.cumsum(0) <= s.tokens)
    need, rows = torch.where(served, need, 0), torch.where(served, rows, 0)
    grown = (at >= kept[:, None]) & (at < (kept + need)[:, None])
    taken = need.sum()
    s.table[grown] = s.free_pages[count - 1 - torch.arange(int(taken), device=pages.device)]
    s.free_count[0] = count - taken
    s.lens.copy_(keep + rows)
    starts = torch.cat([rows.new_zeros(1), rows.cumsum(0)])
    t = torch.arange(s.tokens, device=s.table.device)
    b = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    real = b < rows.numel()
    b = b.clamp(max=rows.numel() - 1)
    position = keep[b] + t - starts[b]
    slots = s.table[b, (position // page).clamp(0, width - 1)].long() * page + position % page
    return [starts.int(), torch.where(real, position, -1).int(), torch.where(real, slots, -1), s.lens, s.table, s.free_pages, s.free_count]


def _places(s):
    """Sequence and position of each real token."""
    t = torch.arange(s.real, device=s.starts.device)
    b = torch.searchsorted(s.starts[1:].long(), t, right=True)
    return b, s.lens[b].long() - s.starts[b + 1].long() + t


def _plain_append(s):
    """Keys in 64 bits: a number next to the border of two codes falls on the side where its exact value lies."""
    b, p = _places(s)
    q, k = s.q[:s.real].float(), s.new_k[:s.real].double()
    if s.q_gamma is not None:
        q, k = _normed(q, s.q_gamma, s.eps), _normed(k, s.k_gamma, s.eps)
    if s.cos_sin is not None:
        q, k = _rotated(q, s.cos_sin[p], s.interleaved), _rotated(k, s.cos_sin[p], s.interleaved)
    page = s.k.size(1)
    pages, at = s.table[b, p // page].long(), p % page
    s.k[pages, at], s.k_scales[pages, at] = _quantized(k, s.most)
    s.v[pages, at], s.v_scales[pages, at] = _quantized(s.new_v[:s.real].float(), s.most)
    out = torch.zeros(s.q.shape, dtype=s.dtype, device=s.q.device)
    out[:s.real] = q.to(s.dtype)
    return [out, _values(s.k, s.k_scales).to(s.dtype), _values(s.v, s.v_scales).to(s.dtype)]


def _plain_attention(s):
    seqs, hq, hk, d = s.lens.numel(), s.q.size(1), s.k.size(2), s.q.size(2)
    group, page = hq // hk, s.k.size(1)
    b, p = _places(s)
    row = torch.arange(s.real, device=s.q.device) - s.starts[b].long()
    # queries as [sequence, key head, row and head of the group, dim]; keys and values gathered as [sequence, key head, key, dim]
    q = s.q.new_zeros((seqs, s.longest_new, hq, d), dtype=torch.float32)
    q[b, row] = s.q[:s.real].float()
    q = q.view(seqs, s.longest_new, hk, group, d).permute(0, 2, 1, 3, 4).reshape(seqs, hk, s.longest_new * group, d)
    j = torch.arange(s.longest, device=s.q.device)
    pages, at = s.table[:, j // page].long(), j % page
    k = _values(s.k[pages, at], s.k_scales[pages, at]).permute(0, 2, 3, 1).contiguous()
    v = _values(s.v[pages, at], s.v_scales[pages, at]).permute(0, 2, 1, 3).contiguous()
    first = s.lens.long() - (s.starts[1:] - s.starts[:-1]).long()
    visible = j <= (first[:, None] + torch.arange(s.longest_new, device=s.q.device))[:, :, None]
    visible = visible & (j < s.lens[:, None, None])
    scores = torch.matmul(q, k).mul_(s.scale).view(seqs, hk, s.longest_new, group, s.longest)
    scores.masked_fill_(~visible[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()   # rows that no sequence of the padded layout has see nothing
    scores = scores.div_(scores.sum(-1, keepdim=True)).view(seqs, hk, s.longest_new * group, s.longest)
    o = torch.matmul(scores, v).view(seqs, hk, s.longest_new, group, d).permute(0, 2, 1, 3, 4).reshape(seqs, s.longest_new, hq, d)
    out = torch.zeros(s.q.shape, dtype=s.dtype, device=s.q.device)
    out[:s.real] = o[b, row].to(s.dtype)
    return out


def run(s):
    if own:
        import torch_dist_ext_amd as tde
        if s.op == "update_pages":
            maps = tde.update_pages(s.table, s.lens, s.new, s.free_pages, s.free_count, s.page, s.tokens, keep_lens=s.keep)
            return [*maps, s.lens, s.table, s.free_pages, s.free_count]
        if s.op == "append_kv_fp4":
            q = tde.append_kv_fp4(s.new_k, s.new_v, s.k, s.k_scales, s.v, s.v_scales, s.table, s.starts, s.lens, cos_sin=s.cos_sin, q=s.q,
                                  q_gamma=s.q_gamma, k_gamma=s.k_gamma, eps=s.eps, interleaved=s.interleaved)
            return [q, tde.unpack_fp4(s.k, s.k_scales, s.dtype), tde.unpack_fp4(s.v, s.v_scales, s.dtype)]
        if s.op == "unpack_fp4":
            return tde.unpack_fp4(s.codes, s.scales, s.dtype)
        return tde.paged_attention_fp4(s.q, s.k, s.k_scales, s.v, s.v_scales, s.table, s.starts, s.lens, s.scale)
    if s.op == "unpack_fp4":
        return _values(s.codes, s.scales).to(s.dtype)
    return {"update_pages": _plain_pages, "append_kv_fp4": _plain_append, "paged_attention_fp4": _plain_attention}[s.op](s)


def work(case):
    page = case["page"]
    if case["op"] == "update_pages":
        new, keep = _lengths(case)
        moved = sum(-(-(a + b) // page) - -(-b // page) for a, b in zip(new, keep))
        rows = sum(new) + case["pad"]
        # lengths read and written, starts; a page that goes back and comes again is read and written twice; a row's position and slot
        return {"bytes": 20 * case["seqs"] + 16 * moved + 12 * rows, "flops": 0}
    e, hk, d = BYTES[case["dtype"]], case["kv_heads"], case["dim"]
    held = d // 2 + d // 32   # bytes of a key
    if case["op"] == "unpack_fp4":
        n = case["pages"] * page * hk
        return {"bytes": n * (held + d * e), "flops": n * d}
    hq = case["heads"]
    new, ctx = _lengths(case)
    t, lens = sum(new), [a + b for a, b in zip(new, ctx)]
    meta = 8 * case["seqs"] + 4
    pages = sum(-(-a // page) for a in lens)
    if case["op"] == "append_kv_fp4":
        # the rows behind the last sequence are only written, as zeros; tokens share pages' entries; the caches are read back as values
        named = sum(-(-a // page) - b // page for a, b in zip(lens, ctx))
        cache = 2 * (pages + 3) * page * hk
        return {"bytes": t * (hq + 2 * hk) * d * e + (t + case["pad"]) * hq * d * e + 2 * t * hk * held + 4 * t * case["rot"] + 4 * named + meta
                + (2 * d * e if case["norm"] else 0) + cache * (held + d * e),
                "flops": t * (hq + 2 * hk) * d * ((4 if case["norm"] else 0) + 4)}
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, ctx))
    return {"bytes": 2 * sum(lens) * hk * held + (2 * t + case["pad"]) * hq * d * e + 4 * pages + meta, "flops": 4 * pairs * hq * d}


# ---- in 64 bits, written apart from the above -------------------------------------------------------------------------------

def _exact_pages(s):
    """One page at a time, with a list as the stack."""
    table, lens, new, keep = (x.cpu().numpy().astype(np.int64) for x in (s.table, s.lens, s.new, s.keep))
    stack, count = s.free_pages.cpu().numpy().copy(), int(s.free_count[0])
    seqs, width = table.shape
    keep = np.clip(keep, 0, lens)
    pages_of = lambda n: -(-int(n) // s.page)  # noqa: E731
    for b in reversed(range(seqs)):
        for i in reversed(range(pages_of(keep[b]), min(width, pages_of(lens[b])))):
            if count < len(stack):
                stack[count] = table[b, i]
                count += 1
    starts, positions, slots = [0], np.full(s.tokens, -1, np.int32), np.full(s.tokens, -1, np.int64)
    at_first, asked, rows_asked = count, 0, 0
    for b in range(seqs):
        more = pages_of(keep[b] + new[b]) - pages_of(keep[b])
        starts.append(starts[-1])
        lens[b] = keep[b]
        if pages_of(keep[b] + new[b]) > width:
            continue
        asked, rows_asked = asked + more, rows_asked + int(new[b])
        if rows_asked > s.tokens or (more and asked > at_first):
            continue
        for i in range(more):
            count -= 1
            table[b, pages_of(keep[b]) + i] = stack[count]
        for i in range(int(new[b])):
            p, t = int(keep[b]) + i, starts[-1] + i
            positions[t], slots[t] = p, table[b, p // s.page] * s.page + p % s.page
        starts[-1] += int(new[b])
        lens[b] += new[b]
    return [np.array(starts, np.int32), positions, slots, lens.astype(np.int32), table.astype(np.int32), stack, np.array([count], np.int32)]


def _turn(x, rows, interleaved):
    """One pair at a time as a complex number times cos + i sin."""
    half = rows.size(-1) // 2
    z = torch.complex(rows[..., :half], rows[..., half:]).unsqueeze(-2)
    y = x.clone()
    if interleaved:
        w = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:-1], half, 2).contiguous()) * z
        y[..., :2 * half] = torch.view_as_real(w).reshape(*x.shape[:-1], 2 * half)
    else:
        w = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * z
        y[..., :half], y[..., half:2 * half] = w.real, w.imag
    return y


def _unit(x, gamma, eps):
    return gamma.double() * x / ((x * x).sum(-1, keepdim=True) / x.size(-1) + eps).sqrt()


def _decoded(codes, scales):
    sign = torch.tensor([1.0, -1.0], dtype=torch.float64, device=codes.device)
    size = torch.tensor(MAGNITUDES, dtype=torch.float64, device=codes.device)
    x = torch.empty(*codes.shape[:-1], codes.size(-1) * 2, dtype=torch.float64, device=codes.device)
    for half, nibble in enumerate((codes & 15, codes >> 4)):
        x[..., half::2] = size[(nibble & 7).long()] * sign[(nibble >> 3).long()]
    return x * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=-1)


def _rounded_to_4_bits(x, most):
    """x in doubles: the nearest of the eight magnitudes, of two as near the one with the even code."""
    blocks = x.view(*x.shape[:-1], -1, 32)
    largest = blocks.abs().amax(-1, keepdim=True)
    power = torch.floor(torch.log2(largest.clamp(min=2.0 ** -1000)))
    power = power - (torch.exp2(power) > largest).double() + (torch.exp2(power + 1) <= largest).double()
    e = (power - 2 + (largest >= 1.75 * torch.exp2(power)).double()).clamp(LEAST_EXPONENT, most)
    t = blocks.abs() * torch.exp2(-e)
    best, off = torch.zeros_like(t), t.clone()
    for code in range(1, 8):
        d = (t - MAGNITUDES[code]).abs()
        better = (d < off) if code % 2 else (d <= off)
        best, off = torch.where(better, MAGNITUDES[code], best), torch.where(better, d, off)
    return (torch.copysign(best, blocks) * torch.exp2(e)).view_as(x)


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "update_pages":
        return _exact_pages(s)
    if s.op == "unpack_fp4":
        return _decoded(s.codes, s.scales)
    new, ctx = _lengths(case)
    page, at = case["page"], 0
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=s.q.device)
    if s.op == "append_kv_fp4":
        k_cache, v_cache = _decoded(s.k, s.k_scales).contiguous(), _decoded(s.v, s.v_scales).contiguous()
    hk = case["kv_heads"]
    group = case["heads"] // hk
    for b, (n, c) in enumerate(zip(new, ctx)):
        rows = slice(at, at + n)
        at += n
        slots = torch.arange(c + n, device=s.q.device)
        pages, slots = s.table[b].long()[slots // page], slots % page
        if s.op == "append_kv_fp4":
            q, k, v = s.q[rows].double(), s.new_k[rows].double(), s.new_v[rows].double().contiguous()
            if case["norm"]:
                q, k = _unit(q, s.q_gamma, s.eps), _unit(k, s.k_gamma, s.eps)
            if case["rot"]:
                q, k = (_turn(x, s.cos_sin[c:c + n].double(), s.interleaved) for x in (q, k))
            out[rows] = q
            k_cache[pages[c:], slots[c:]] = _rounded_to_4_bits(k.contiguous(), s.most)
            v_cache[pages[c:], slots[c:]] = _rounded_to_4_bits(v, s.most)
            continue
        for h in range(hk):
            k, v = (_decoded(x[pages, slots, h], y[pages, slots, h]) for x, y in ((s.k, s.k_scales), (s.v, s.v_scales)))
            for i in range(group):
                logits = s.q[rows, h * group + i].double() @ k.t().contiguous() * s.scale
                logits += torch.full_like(logits, -math.inf).triu_(c + 1)
                out[rows, h * group + i] = torch.softmax(logits, dim=-1) @ v
    return [out, k_cache, v_cache] if s.op == "append_kv_fp4" else out
