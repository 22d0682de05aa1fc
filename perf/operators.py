"""The operators of an attention block that follow the fused norm on one rank, in their plain form and through the package.

  int8_linear      codes and scales as allreduce_rms_quant(QUANT_INT8_TOKEN) emits them, times an int8 weight with a scale a channel
  qk_norm_rope     RMSNorm of every query and key head and the position rotation
  append_kv        new keys (rotated, optionally normed) and values of a ragged batch into a paged cache, its queries beside them
  paged_attention  the new tokens' queries over the paged cache, causally; one new token a sequence is a decode step

The lengths of a batch are part of the case (`mix` seeds them), so that the work is known; page tables and contents come
from the inputs' seed.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
MOST_FLOPS = 4.12e11   # the largest listed case's
MOST_BYTES = 1.08e9    # the longest listed decode step's
MOST_SCORES = 1.07e9   # scores that the plain form of the attention holds at once: the largest listed chunk's


def _linear(tokens, k, n, out, bias=False, **name):
    return dict(op="int8_linear", tokens=tokens, k=k, n=n, dtype=out, bias=bias, **name)


def _norm_rope(tokens, heads, kv_heads, dim, rot, dtype, interleaved=False, **name):
    return dict(op="qk_norm_rope", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, dtype=dtype,
                interleaved=interleaved, **name)


def _batch(op, seqs, new, ctx, heads, kv_heads, dim, page, dtype, ragged=True, pad=0, mix=1, **more):
    """seqs sequences of up to `new` new tokens each behind up to `ctx` cached ones (exactly so many where not ragged), `pad`
    rows behind the last sequence as a captured step of a fixed size has them."""
    return dict(op=op, seqs=seqs, new=new, ctx=ctx, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, ragged=ragged,
                pad=pad, mix=mix, **more)


def listed():
    return [
        # one token of one sequence through a rank's share of the query/key/value projection: launch and latency
        _linear(1, 8192, 1280, "bf16", name="linear_1x8192x1280"),
        # a decode step of 64 sequences: the weight's bytes
        _linear(64, 5120, 7168, "f16", name="linear_64x5120x7168"),
        # odd sizes: a ragged number of tokens, rows that do not begin on 16 bytes, channels that fill no tile, fp32 and a bias
        _linear(1257, 5000, 1100, "f32", bias=True, name="linear_1257x5000x1100_f32"),
        # prefill of 2048 tokens: matrix instructions
        _linear(2048, 8192, 8192, "bf16", name="linear_2048x8192x8192"),
        # a decode step of 64 sequences on one of eight ranks
        _norm_rope(64, 8, 1, 128, 128, "bf16", name="norm_rope_64x9"),
        # a long prefill with all heads of a model on one GPU
        _norm_rope(8192, 32, 8, 128, 128, "bf16", name="norm_rope_8192x40"),
        # a decode step of 128 sequences: norm, rotation and append in one call
        _batch("append_kv", 128, 1, 4096, 8, 1, 128, 64, "bf16", norm=True, rot=128, interleaved=False, name="append_128x1"),
        # chunks of four sequences, half of a head's channels rotated in adjacent pairs, no norm
        _batch("append_kv", 4, 2048, 2048, 32, 8, 128, 16, "f16", ragged=False, norm=False, rot=64, interleaved=True,
               name="append_4x2048_f16"),
        # a decode step of 64 sequences of very different lengths: the cache's bytes
        _batch("paged_attention", 64, 1, 8192, 32, 8, 128, 64, "bf16", name="decode_64x8192"),
        # one long sequence on one of eight ranks: one key head, one token
        _batch("paged_attention", 1, 1, 131071, 8, 1, 128, 128, "bf16", ragged=False, name="decode_1x131072"),
        # a chunk of 4096 tokens behind 4096 cached ones: matrix instructions
        _batch("paged_attention", 1, 4096, 4096, 32, 8, 128, 64, "bf16", ragged=False, name="chunk_4096_of_8192"),
        # a batch that mixes short chunks and long ones, small heads and small pages, padded
        _batch("paged_attention", 24, 512, 2048, 12, 4, 64, 16, "f16", pad=37, mix=3, name="mixed_24x512_f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["int8_linear", "int8_linear", "qk_norm_rope", "append_kv", "paged_attention", "paged_attention"])
        if op == "int8_linear":
            k = _log(rng, 64, 8192)
            if rng.random() < 0.8:   # whole 8 bytes: what the fused norm's 2-byte rows give
                k = max(8, k // 8 * 8)
            c = _linear(_log(rng, 1, 8192), k, _log(rng, 48, 8192), rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.3)
        elif op == "qk_norm_rope":
            dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
            kv_heads = rng.choice([1, 2, 4, 5, 8])
            c = _norm_rope(_log(rng, 1, 16384), kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads, dim, rng.choice([dim, dim, dim // 2]),
                           rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.3)
        else:
            dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
            kv_heads = rng.choice([1, 2, 4, 5, 8])
            heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
            kind = rng.choice(["decode", "chunk", "mixed"])
            seqs = {"decode": _log(rng, 1, 256), "chunk": rng.randint(1, 3), "mixed": rng.randint(2, 32)}[kind]
            new = {"decode": 1, "chunk": _log(rng, 16, 4096), "mixed": _log(rng, 2, 1024)}[kind]
            ctx = _log(rng, 1, 131072 if kind == "decode" else 16384)
            page, pad = rng.choice([8, 16, 16, 24, 64, 128]), rng.choice([0, 0, rng.randint(1, 64)])
            ragged, mix = rng.random() < 0.7, rng.randint(1, 1 << 20)
            if op == "append_kv":
                c = _batch(op, seqs, new, ctx, heads, kv_heads, dim, page, rng.choice(["bf16", "bf16", "f16", "f32"]), ragged, pad, mix,
                           norm=rng.random() < 0.5, rot=rng.choice([0, dim, dim, dim // 2]), interleaved=rng.random() < 0.3)
            else:
                c = _batch(op, seqs, new, ctx, heads, kv_heads, dim, page, rng.choice(["bf16", "bf16", "f16"]), ragged, pad, mix)
            if seqs * (new + ctx) * kv_heads * dim * 4 > 2e9 or heads * seqs * new * (new + ctx) > MOST_SCORES:
                continue
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return c


def _lengths(case):
    """New tokens and cached ones of each sequence."""
    if not case["ragged"]:
        return [case["new"]] * case["seqs"], [case["ctx"]] * case["seqs"]
    rng = random.Random(case["mix"])
    return ([rng.randint(1, case["new"]) for _ in range(case["seqs"])], [rng.randint(0, case["ctx"]) for _ in range(case["seqs"])])


class State:
    """One call's inputs and what a program keeps between calls: weights, tables, caches."""


def _gamma(n, g, dev, dtype):
    return (torch.rand(n, generator=g, device=dev) + 0.5).to(dtype)


def _cos_sin(positions, rot, dev):
    """fp32 rows of rot/2 cosines and rot/2 sines, the angles in doubles."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
    a = torch.arange(positions, device=dev, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    s = State()
    s.op, s.dtype = case["op"], dtype

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype)

    if s.op == "int8_linear":
        t, k, n = case["tokens"], case["k"], case["n"]
        # a normed row quantized by its largest magnitude, about four standard deviations out; weights alike
        s.codes = torch.randn((t, k), generator=g, device=dev).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        s.scales = (torch.rand(t, generator=g, device=dev) + 0.5) * (4 / 127)
        s.weight = torch.randn((n, k), generator=g, device=dev).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        s.weight_scales = (torch.rand(n, generator=g, device=dev) + 0.5) * (4 / 127 / math.sqrt(k))
        s.bias = torch.randn(n, generator=g, device=dev) if case["bias"] else None
        return s
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    s.eps, s.interleaved = 1e-6, case.get("interleaved", False)
    if s.op == "qk_norm_rope":
        t = case["tokens"]
        # queries and keys are column ranges of one projection's output
        qkv = randn(t, hq + 2 * hk, d)
        s.q, s.k = qkv[:, :hq], qkv[:, hq:hq + hk]
        s.q_gamma, s.k_gamma = _gamma(d, g, dev, dtype), _gamma(d, g, dev, dtype)
        s.positions = torch.randint(0, 32768, (t,), generator=g, device=dev)
        s.cos_sin = _cos_sin(32768, case["rot"], dev)
        return s
    new, ctx = _lengths(case)
    lens = [a + b for a, b in zip(new, ctx)]
    starts = [0]
    for a in new:
        starts.append(starts[-1] + a)
    s.real, s.longest_new, s.longest = starts[-1], max(new), max(lens)
    t, page = s.real + case["pad"], case["page"]
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
    s.k_cache, s.v_cache = randn(sum(need) + 3, page, hk, d), randn(sum(need) + 3, page, hk, d)
    if s.op == "append_kv":
        qkv = randn(t, hq + 2 * hk, d)
        s.q, s.k, s.v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        s.q_gamma = _gamma(d, g, dev, dtype) if case["norm"] else None
        s.k_gamma = _gamma(d, g, dev, dtype) if case["norm"] else None
        s.cos_sin = _cos_sin(s.longest, case["rot"], dev) if case["rot"] else None
    else:
        s.q = randn(t, hq, d)
        s.scale = d ** -0.5
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------

def _normed(x, gamma, eps):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * gamma.float()


def _rotated(x, rows, interleaved):
    """x [T, heads, dim] in fp32, rows [T, rot] of cosines and sines."""
    half = rows.size(1) // 2
    c, s = rows[:, None, :half], rows[:, None, half:]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _plain_linear(s):
    y = s.codes.float() @ s.weight.float().t()
    y = y * s.scales[:, None] * s.weight_scales
    return (y if s.bias is None else y + s.bias).to(s.dtype)


def _plain_norm_rope(s):
    rows = s.cos_sin[s.positions]
    return [_rotated(_normed(s.q, s.q_gamma, s.eps), rows, s.interleaved).to(s.dtype),
            _rotated(_normed(s.k, s.k_gamma, s.eps), rows, s.interleaved).to(s.dtype)]


def _places(s):
    """Sequence and position of each real token."""
    t = torch.arange(s.real, device=s.starts.device)
    b = torch.searchsorted(s.starts[1:].long(), t, right=True)
    return b, s.lens[b].long() - s.starts[b + 1].long() + t


def _plain_append(s):
    b, p = _places(s)
    q, k = s.q[:s.real], s.k[:s.real]
    q, k = (q.float(), k.float()) if s.q_gamma is None else (_normed(q, s.q_gamma, s.eps), _normed(k, s.k_gamma, s.eps))
    if s.cos_sin is not None:
        rows = s.cos_sin[p]
        q, k = _rotated(q, rows, s.interleaved), _rotated(k, rows, s.interleaved)
    page = s.k_cache.size(1)
    pages, at = s.table[b, p // page].long(), p % page
    s.k_cache[pages, at] = k.to(s.dtype)
    s.v_cache[pages, at] = s.v[:s.real]
    out = torch.zeros(s.q.shape, dtype=s.dtype, device=s.q.device)
    out[:s.real] = q.to(s.dtype)
    return [out, s.k_cache, s.v_cache]


def _plain_attention(s):
    seqs, hq, hk, d = s.lens.numel(), s.q.size(1), s.k_cache.size(2), s.q.size(2)
    group, page = hq // hk, s.k_cache.size(1)
    b, p = _places(s)
    row = torch.arange(s.real, device=s.q.device) - s.starts[b].long()
    # queries as [sequence, key head, row and head of the group, dim]; keys and values gathered as [sequence, key head, key, dim]
    q = s.q.new_zeros((seqs, s.longest_new, hq, d), dtype=torch.float32)
    q[b, row] = s.q[:s.real].float()
    q = q.view(seqs, s.longest_new, hk, group, d).permute(0, 2, 1, 3, 4).reshape(seqs, hk, s.longest_new * group, d)
    j = torch.arange(s.longest, device=s.q.device)
    pages, at = s.table[:, j // page].long(), j % page
    k = s.k_cache[pages, at].permute(0, 2, 3, 1).float().contiguous()
    v = s.v_cache[pages, at].permute(0, 2, 1, 3).float().contiguous()
    first = s.lens.long() - (s.starts[1:] - s.starts[:-1]).long()
    visible = j <= (first[:, None] + torch.arange(s.longest_new, device=s.q.device))[:, :, None]
    visible = visible & (j < s.lens[:, None, None])
    scores = torch.matmul(q, k).mul_(s.scale).view(seqs, hk, s.longest_new, group, s.longest)
    scores.masked_fill_(~visible[:, None, :, None, :], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    scores = scores.div_(scores.sum(-1, keepdim=True)).view(seqs, hk, s.longest_new * group, s.longest)
    o = torch.matmul(scores, v).view(seqs, hk, s.longest_new, group, d).permute(0, 2, 1, 3, 4).reshape(seqs, s.longest_new, hq, d)
    out = torch.zeros(s.q.shape, dtype=s.dtype, device=s.q.device)
    out[:s.real] = o[b, row].to(s.dtype)
    return out


def run(s):
    if own:
        import torch_dist_ext_amd as tde
        if s.op == "int8_linear":
            return tde.int8_linear(s.codes, s.scales, s.weight, s.weight_scales, s.bias, s.dtype)
        if s.op == "qk_norm_rope":
            return tde.qk_norm_rope(s.q, s.k, s.q_gamma, s.k_gamma, s.eps, s.positions, s.cos_sin, s.interleaved)
        if s.op == "append_kv":
            q = tde.append_kv(s.k, s.v, s.k_cache, s.v_cache, s.table, s.starts, s.lens, cos_sin=s.cos_sin, q=s.q, q_gamma=s.q_gamma,
                              k_gamma=s.k_gamma, eps=s.eps, interleaved=s.interleaved)
            return [q, s.k_cache, s.v_cache]
        return tde.paged_attention(s.q, s.k_cache, s.v_cache, s.table, s.starts, s.lens, s.scale)
    return {"int8_linear": _plain_linear, "qk_norm_rope": _plain_norm_rope, "append_kv": _plain_append,
            "paged_attention": _plain_attention}[s.op](s)


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "int8_linear":
        t, k, n = case["tokens"], case["k"], case["n"]
        return {"bytes": t * k + n * k + 4 * t + 4 * n + (4 * n if case["bias"] else 0) + t * n * e, "flops": 2 * t * k * n}
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "qk_norm_rope":
        t = case["tokens"]
        # rows in and out, the gammas, a position and a row of the rotation's table for each token
        return {"bytes": 2 * t * (hq + hk) * d * e + 2 * d * e + t * (8 + 4 * case["rot"]), "flops": t * (hq + hk) * d * 7}
    new, ctx = _lengths(case)
    t, lens = sum(new), [a + b for a, b in zip(new, ctx)]
    meta = 8 * case["seqs"] + 4
    if case["op"] == "append_kv":
        # the rows behind the last sequence are only written, as zeros; tokens share pages' entries
        pages = sum(-(-a // case["page"]) - b // case["page"] for a, b in zip(lens, ctx))
        return {"bytes": 2 * t * (hq + 2 * hk) * d * e + case["pad"] * hq * d * e + 4 * t * case["rot"] + 4 * pages + meta
                + (2 * d * e if case["norm"] else 0),
                "flops": t * (hq + hk) * d * ((4 if case["norm"] else 0) + 3)}
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, ctx))
    pages = sum(-(-a // case["page"]) for a in lens)
    return {"bytes": 2 * sum(lens) * hk * d * e + (2 * t + case["pad"]) * hq * d * e + 4 * pages + meta, "flops": 4 * pairs * hq * d}


# ---- in 64 bits, written apart from the above -------------------------------------------------------------------------------

def _turn(x, angles_row, interleaved):
    """One pair at a time as a complex number times cos + i sin."""
    half = angles_row.size(-1) // 2
    z = torch.complex(angles_row[..., :half], angles_row[..., half:]).unsqueeze(-2)
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


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "int8_linear":
        y = torch.mm(s.codes.double(), s.weight.double().t().contiguous())   # whole numbers below 2^53: no rounding
        y = y * torch.outer(s.scales.double(), s.weight_scales.double())
        return y if s.bias is None else y + s.bias.double()
    if s.op == "qk_norm_rope":
        rows = s.cos_sin.double()[s.positions]
        return [_turn(_unit(x.double(), gamma, s.eps), rows, s.interleaved) for x, gamma in ((s.q, s.q_gamma), (s.k, s.k_gamma))]
    new, ctx = _lengths(case)
    page, at = case["page"], 0
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=s.q.device)
    if s.op == "append_kv":
        k_cache, v_cache = s.k_cache.double(), s.v_cache.double()
    for b, (n, c) in enumerate(zip(new, ctx)):
        rows = slice(at, at + n)
        at += n
        slots = torch.arange(c + n, device=s.q.device)
        slots = s.table[b].long()[slots // page] * page + slots % page
        if s.op == "append_kv":
            q, k = s.q[rows].double(), s.k[rows].double()
            if case["norm"]:
                q, k = _unit(q, s.q_gamma, s.eps), _unit(k, s.k_gamma, s.eps)
            if case["rot"]:
                q, k = (_turn(x, s.cos_sin[c:c + n].double(), s.interleaved) for x in (q, k))
            out[rows] = q
            k_cache.view(-1, *k.shape[1:])[slots[c:]] = k
            v_cache.view(-1, *k.shape[1:])[slots[c:]] = s.v[rows].double()
            continue
        hk = case["kv_heads"]
        group = case["heads"] // hk
        for h in range(hk):
            k, v = (x.view(-1, hk, x.size(-1))[slots, h].double() for x in (s.k_cache, s.v_cache))
            for i in range(group):
                logits = s.q[rows, h * group + i].double() @ k.t().contiguous() * s.scale
                logits += torch.full_like(logits, -math.inf).triu_(c + 1)
                out[rows, h * group + i] = torch.softmax(logits, dim=-1) @ v
    return [out, k_cache, v_cache] if s.op == "append_kv" else out
