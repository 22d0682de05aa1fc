"""The attention block's operators from their definitions, in doubles on the CPU, and how far a result in T may be off.

Every bound counts roundings: half a step of T (`finfo.eps / 2` of the value) for each rounding to T, 2^-24 for each in fp32."""
import math

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half a step among T's subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def assert_close(got, want, bound, what=""):
    """`want` and `bound` in doubles; where want is not finite, got is the same (NaN for NaN)."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    same = (torch.isnan(got) & torch.isnan(want)) | (got == want)
    off = (got - want).abs()
    ok = torch.where(fine, off <= bound, same)
    if not bool(ok.all()):
        bad = (~ok).nonzero()
        at = tuple(bad[0].tolist())
        raise AssertionError("%s: %d of %d wrong, first at %s: got %r, want %r, bound %r" % (
            what, bad.size(0), ok.numel(), at, got[at].item(), want[at].item(), torch.as_tensor(bound).expand(want.shape)[at].item()))


# ---- int8 product ----

def int8_linear(codes, scales, weight, weight_scales, bias, dtype):
    total = codes.double() @ weight.double().t()   # whole numbers below 2^31
    y = total * scales.double().reshape(*codes.shape[:-1], 1) * weight_scales.double()
    want = y if bias is None else y + bias.double()
    # float(sum), the scales' product, their product: 3 roundings of y; the addition: one of the result
    bound = y.abs() * 3.01 * U32 + want.abs() * (U32 + half_step(dtype)) * 1.01 + smallest(dtype)
    limit = torch.finfo(dtype).max
    over = want.abs() > limit * (1 + half_step(dtype))
    return torch.where(over, torch.sign(want) * math.inf, want), bound


# ---- norm and rotation ----

def norm_rope(x, gamma, eps, rows, interleaved, dtype):
    """x [T, heads, dim]; gamma [dim] or None; rows [T, rot] or None (NaN rows: positions outside the table)."""
    dim = x.size(-1)
    u = x.double()
    if gamma is not None:
        u = u / (u.square().mean(-1, keepdim=True) + eps).sqrt() * gamma.double()
    # dim squares added in fp32 (the root halves what that costs), divided, rooted, inverted, two products
    rel = (dim / 2 + 6) * U32 if gamma is not None else 0.0
    want, size = u.clone(), u.abs()
    if rows is not None and rows.size(-1):
        half = rows.size(-1) // 2
        c, s = rows[:, None, :half].double(), rows[:, None, half:].double()
        a_at = slice(0, 2 * half, 2) if interleaved else slice(0, half)
        b_at = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
        a, b = u[..., a_at], u[..., b_at]
        want[..., a_at], want[..., b_at] = a * c - b * s, b * c + a * s
        size = size.clone()
        size[..., a_at], size[..., b_at] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
        rel += 2 * U32
    bound = size * rel * 1.01 + want.abs() * half_step(dtype) * 1.01 + smallest(dtype)
    return want, bound


# ---- paged batches ----

class Batch:
    """A ragged batch: new rows and keys of each sequence, pages in no order, rows behind the last sequence."""

    def __init__(self, new, lens, page_size, extra_pages=2, pad=0, seed=0, table_pages=None):
        g = torch.Generator().manual_seed(seed)
        self.new, self.lens, self.page, self.pad = list(new), list(lens), page_size, pad
        need = [-(-max(0, n) // page_size) for n in lens]
        self.pages = sum(need) + extra_pages
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        width = max(need + [1]) if table_pages is None else table_pages
        self.table = torch.full((len(new), width), -7, dtype=torch.int32)
        at = 0
        for b, m in enumerate(need):
            self.table[b, :min(m, width)] = order[at:at + m][:width]
            at += m
        self.starts = torch.zeros(len(new) + 1, dtype=torch.int32)
        if new:
            self.starts[1:] = torch.tensor(new, dtype=torch.int32).cumsum(0)
        self.kv_lens = torch.tensor(self.lens, dtype=torch.int32)
        self.tokens = int(self.starts[-1]) + pad

    def rows(self):
        """(token, sequence, position) of every row of a sequence."""
        t = 0
        for b, (n, length) in enumerate(zip(self.new, self.lens)):
            for i in range(n):
                yield t, b, max(0, length) - n + i
                t += 1

    def page_of(self, b, position):
        at = position // self.page
        if at >= self.table.size(1):
            return None
        page = int(self.table[b, at])
        return page if 0 <= page < self.pages else None

    def on(self, device):
        return [x.to(device) for x in (self.table, self.starts, self.kv_lens)]


def append(batch, k_want, v, k_cache, v_cache):
    """The caches after the call: k_want [T, heads, dim] in doubles; caches [pages, page_size, heads, dim].  Returns (keys in doubles,
    values, which slots were written)."""
    keys, values = k_cache.double().clone(), v_cache.clone()
    written = torch.zeros(k_cache.shape[:2], dtype=torch.bool)
    token_of = torch.full(k_cache.shape[:2], -1, dtype=torch.long)
    for t, b, p in batch.rows():
        if p < 0:
            continue
        page = batch.page_of(b, p)
        if page is None:
            continue
        keys[page, p % batch.page], values[page, p % batch.page] = k_want[t], v[t]
        written[page, p % batch.page] = True
        token_of[page, p % batch.page] = t
    return keys, values, written, token_of


def attention(batch, q, k_cache, v_cache, scale):
    """Rows one by one: what a row does not see is never touched.  Rows behind the last sequence are zeros."""
    dtype = q.dtype
    heads, kv_heads, dim = q.size(1), k_cache.size(2), q.size(2)
    group = heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    h = half_step(dtype)
    gathered = {}
    for t, b, p in batch.rows():
        if p < 0:
            continue
        if b not in gathered:
            lost = next((j for j in range(max(0, batch.lens[b])) if batch.page_of(b, j) is None), None)
            n = max(0, batch.lens[b]) if lost is None else lost
            j = torch.arange(n)
            pages = batch.table[b].long()[j // batch.page] if n else j
            gathered[b] = (lost, k_cache[pages, j % batch.page].double(), v_cache[pages, j % batch.page].double())
        lost, keys, values = gathered[b]
        if lost is not None and p >= lost:
            out[t] = math.nan
            continue
        n = p + 1
        for kv in range(kv_heads):
            qs = q[t, kv * group:(kv + 1) * group].double()
            k, v = keys[:n, kv], values[:n, kv]
            s = qs @ k.t() * scale
            w = torch.softmax(s, dim=-1)
            o = torch.stack([(w[i][:, None] * v).sum(0) for i in range(group)])
            out[t, kv * group:(kv + 1) * group] = o
            # a score: dim products added, scaled, shifted; it enters as an exponent.  Twice: numerator and sum.
            reach = (qs.abs() @ k.abs().t()).amax(-1, keepdim=True) * scale
            rel = 2 * (reach * (dim + 6) * U32 + (n + 16) * U32)
            size = w @ v.abs().nan_to_num(0.0, 0.0, 0.0)
            # every weight is rounded to T, subnormal ones by an absolute half step (the largest weight is 1, so the sum is at least 1)
            bound[t, kv * group:(kv + 1) * group] = (size * (h + rel) * 1.02 + o.abs() * (h + rel) * 1.02 + smallest(dtype)
                                                     + smallest(dtype) * v.abs().nan_to_num(0.0, 0.0, 0.0).sum(0))
    return out, bound


def attention_at_once(batch, q, k_cache, v_cache, scale):
    """The same for long chunks, on the tensors' device: products over a sequence's rows.  Values that are not finite reach exactly the
    rows whose keys include them (every weight stays above zero here); keys are finite wherever a row sees them."""
    dtype, device = q.dtype, q.device
    heads, kv_heads, dim = q.size(1), k_cache.size(2), q.size(2)
    group, h = heads // kv_heads, half_step(q.dtype)
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device=device), torch.zeros(q.shape, dtype=torch.float64, device=device)
    at = 0
    for b, (new, length) in enumerate(zip(batch.new, batch.lens)):
        first, at = at, at + new
        length = max(0, length)
        if not new:
            continue
        lost = next((p * batch.page for p in range(-(-length // batch.page)) if batch.page_of(b, p * batch.page) is None), length)
        j = torch.arange(lost)
        pages = batch.table[b].long()[j // batch.page].to(device)
        positions = torch.arange(length - new, length, device=device)
        sees = torch.arange(lost, device=device)[None, :] <= positions[:, None]
        counts = (positions + 1).double()[:, None]
        for kv in range(kv_heads):
            k = k_cache[pages, (j % batch.page).to(device), kv].double()
            v = v_cache[pages, (j % batch.page).to(device), kv].double()
            k = torch.where(sees.any(0)[:, None], k, 0.0)
            finite = v.nan_to_num(0.0, 0.0, 0.0)
            kt, kt_abs = k.t().contiguous(), k.abs().t().contiguous()
            mask = sees.double()
            nan, up, down = ((mask @ x.double()) > 0 for x in (v.isnan(), v == math.inf, v == -math.inf))
            beyond = mask @ finite.abs()
            for head in range(kv * group, (kv + 1) * group):
                rows = q[first:at, head].double()
                s = torch.where(sees, rows @ kt * scale, -math.inf)
                w = torch.where(sees.any(1)[:, None], torch.softmax(s, dim=-1), 0.0)
                assert bool((w[sees] > 0).all())
                o = w @ finite
                reach = torch.where(sees, rows.abs() @ kt_abs, 0.0).amax(-1, keepdim=True) * scale
                rel = 2 * (reach * (dim + 6) * U32 + (counts + 16) * U32)
                bound[first:at, head] = (w @ finite.abs() + o.abs()) * (h + rel) * 1.02 + smallest(dtype) + smallest(dtype) * beyond
                bound[first:at, head][positions < 0] = 0.0
                o = torch.where(up, math.inf, torch.where(down, -math.inf, o))
                o[nan | (up & down)] = math.nan
                o[positions >= lost] = math.nan
                o[positions < 0] = 0.0
                out[first:at, head] = o
    return out.cpu(), bound.nan_to_num(0.0).cpu()
