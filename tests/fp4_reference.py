"""A paged cache in 4 bits, from its definition in doubles on the CPU: what codes and scales stand for, how numbers are rounded, whose pages are whose."""
import math

import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def decode(codes, scales):
    """[..., dim / 2] and [..., dim / 32] bytes as doubles [..., dim]."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=torch.float64)
    x = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], dim=-1).flatten(-2)
    unit = torch.exp2(scales.double() - 127)
    unit[scales == 255] = math.nan
    return x * unit.repeat_interleave(32, dim=-1)


def encode(x, most):
    """x [..., dim] in doubles -> (codes, scales), one number at a time from the nearest of sixteen, of two as near the one with an even code."""
    blocks = x.reshape(-1, 32)
    codes, scales = torch.zeros(blocks.shape, dtype=torch.uint8), torch.zeros(blocks.size(0), dtype=torch.uint8)
    largest = blocks.abs().amax(1)
    finite = torch.isfinite(blocks).all(1)
    fraction, exponent = torch.frexp(torch.where(finite, largest, 0.0))
    e = (exponent - 1 - 2 + (2 * fraction >= 1.75).int()).clamp(-125, most)
    e[finite & (largest == 0)] = -125
    t = blocks.abs() / torch.exp2(e.double())[:, None]
    sizes = torch.tensor(MAGNITUDES, dtype=torch.float64)
    off = (t[..., None] - sizes).abs()
    nearest = off.amin(-1, keepdim=True)
    even_first = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])
    codes = even_first[(off == nearest)[..., even_first].int().argmax(-1)].to(torch.uint8)
    codes |= torch.signbit(blocks).to(torch.uint8) << 3
    codes[~finite] = 0
    scales = torch.where(finite, e + 127, 255).to(torch.uint8)
    codes = codes.reshape(x.shape)
    return codes[..., 0::2] | codes[..., 1::2] << 4, scales.reshape(*x.shape[:-1], x.size(-1) // 32)


def most_exponent(dtype):
    return 13 if dtype == torch.float16 else 125


def random_cache(shape, dim, seed, spread=1.0):
    """Codes and scales of random numbers for `shape` heads."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((*shape, dim), generator=g).double() * spread
    return encode(x, 125)


def as_read(codes, scales, dtype):
    """The numbers of `dtype` that an attention reads, in doubles: blocks whose 6 is no number of fp16 are NaN there."""
    if dtype == torch.float16:
        scales = torch.where(scales > 127 + 13, 255, scales)
    return decode(codes, scales).to(dtype).double()


class Pages:
    """The stack of free pages and the sequences' lists, moved one page at a time."""

    def __init__(self, table, lens, free, count):
        self.table, self.lens, self.free, self.count = table.clone().long(), lens.clone().long(), free.clone().long(), int(count)

    def step(self, new, page, tokens, keep=None):
        seqs, width = self.table.shape
        room = len(self.free)
        count = min(max(self.count, 0), room)
        pages_of = lambda n: -(-int(n) // page)  # noqa: E731
        lens = [max(0, int(n)) for n in self.lens]
        keeps = lens if keep is None else [min(max(0, int(k)), n) for k, n in zip(keep, lens)]
        back = [int(self.table[b, i]) for b in range(seqs) for i in range(min(pages_of(keeps[b]), width), min(pages_of(lens[b]), width))]
        for page_number in reversed(back):
            if count < room:
                self.free[count] = page_number
                count += 1
        there, asked, rows_asked = count, 0, 0
        starts, positions, slots = [0], [-1] * tokens, [-1] * tokens
        for b in range(seqs):
            more, had = max(0, int(new[b])), min(pages_of(keeps[b]), width)
            starts.append(starts[-1])
            self.lens[b] = keeps[b]
            if pages_of(keeps[b] + more) > width or keeps[b] + more > 0x7fffffff:
                continue
            need = pages_of(keeps[b] + more) - had if more else 0
            asked, rows_asked = asked + need, rows_asked + more
            if rows_asked > tokens or (need and asked > there):
                continue
            for i in range(need):
                count -= 1
                self.table[b, had + i] = self.free[count]
            for i in range(more):
                p = keeps[b] + i
                positions[starts[-1]] = p
                slots[starts[-1]] = int(self.table[b, p // page]) * page + p % page
                starts[-1] += 1
            self.lens[b] = keeps[b] + more
        self.count = count
        return torch.tensor(starts), torch.tensor(positions, dtype=torch.long), torch.tensor(slots, dtype=torch.long)
