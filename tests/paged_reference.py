"""The paged cache's operators in 64 bits on the CPU, one token at a time, and inputs for them."""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

from exp3_amd import paged

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def four_bit(x):
    """[..., D] float64 -> the value that its 4-bit row stands for: the scale of each 32 is the
    power of two that puts the largest into [3.5, 7), values go to the nearest grid point, the
    even one at ties."""
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(top)[1] - 1                     # floor(log2 top)
    exponent = exponent + (top >= torch.ldexp(torch.tensor(1.75, dtype=torch.float64), exponent))
    step = torch.ldexp(torch.ones((), dtype=torch.float64), (exponent - 2).clamp(-125, 125))
    off = ((x.abs() / step)[..., None] - GRID).abs()
    near = off.amin(-1, keepdim=True)
    even = (off == near) & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.float().argmax(-1), (off == near).float().argmax(-1))
    out = torch.copysign(GRID[code] * step, x)
    return torch.where(torch.isfinite(top), out, math.nan).flatten(-2)


def rotated(x, cos, sin, interleaved=False):
    """[..., D] float64, the first 2 x cos.shape[-1] dims."""
    half = cos.shape[-1]
    pair = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else \
        (slice(0, half), slice(half, 2 * half))
    a, b = x[..., pair[0]], x[..., pair[1]]
    out = x.clone()
    out[..., pair[0]] = a * cos - b * sin
    out[..., pair[1]] = b * cos + a * sin
    return out


def live_position(s, b, i):
    start = int(s.starts[b])
    p = start + i
    live = start >= 0 and (s.counts is None or i < int(s.counts[b])) \
        and p < s.table.shape[1] * s.page
    return p if live else None


def place(s, b, p):
    """(page, slot) of a position or None."""
    page = int(s.table[b, p // s.page])
    return (page, p % s.page) if 0 <= page < s.pages else None


def make(seed, batch, tokens, q_heads, kv_heads, dim, page, width, starts, counts=None, bits=16,
         rotary=None, sharp=1.0, spare=2):
    """A call's arguments on the CPU and a cache with every slot filled (keys "held")."""
    gen = torch.Generator().manual_seed(seed)

    def draw(*shape):
        return torch.randn(*shape, generator=gen).to(torch.bfloat16)

    pages = batch * width + spare
    s = SimpleNamespace(batch=batch, tokens=tokens, page=page, pages=pages, bits=bits)
    s.table = torch.randperm(pages, generator=gen)[:batch * width].view(batch, width).int()
    s.starts = torch.tensor(starts, dtype=torch.int32)
    s.counts = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    s.q, s.k, s.v = (draw(batch, tokens, h, dim) for h in (q_heads, kv_heads, kv_heads))
    s.q = (s.q.float() * sharp).to(torch.bfloat16)
    s.rope = paged.rope_table(width * page, dim if rotary is None else rotary)
    s.held = [draw(pages, kv_heads, page, dim) for _ in range(2)]
    if bits == 4:       # any bytes and scales of a sensible size
        s.raw = [torch.randint(0, 256, (pages, kv_heads, page, dim // 2), generator=gen,
                               dtype=torch.uint8) for _ in range(2)]
        s.scales = [torch.randint(124, 129, (pages, kv_heads, page, dim // 32), generator=gen,
                                  dtype=torch.uint8) for _ in range(2)]
        s.held = [values(r, c) for r, c in zip(s.raw, s.scales)]
    return s


def values(raw, scales):
    """4-bit pages as float64 values."""
    code = torch.stack((raw & 15, raw >> 4), -1).flatten(-2).long()
    size = torch.ldexp(torch.ones((), dtype=torch.float64), scales.int() - 127)
    size = torch.where(scales == 255, math.nan, size)
    signed = torch.cat((GRID, -GRID))[code]
    return (signed.unflatten(-1, (-1, 32)) * size[..., None]).flatten(-2)


def on_gpu(s, four=None):
    """The same call on the GPU: (cache, table, starts, counts)."""
    if s.bits == 4:
        cache = paged.PagedCache(*(x.cuda() for x in s.raw + s.scales))
    else:
        cache = paged.PagedCache(*(x.cuda() for x in s.held))
    return cache, s.table.cuda(), s.starts.cuda(), None if s.counts is None else s.counts.cuda()


def contents(cache):
    """A cache's pages as float64 on the CPU."""
    if cache.four_bit:
        return [values(cache.key_pages.cpu(), cache.key_scales.cpu()),
                values(cache.value_pages.cpu(), cache.value_scales.cpu())]
    return [cache.key_pages.double().cpu(), cache.value_pages.double().cpu()]


def append(s, rope=True, interleaved=False):
    """(rotated q, rotated k, key pages, value pages) in float64; pages of a bf16 cache hold the
    unrounded rows."""
    q, k = s.q.double().clone(), s.k.double().clone()
    pages = [x.double().clone() for x in s.held]
    for b in range(s.batch):
        for i in range(s.tokens):
            p = live_position(s, b, i)
            if p is None:
                q[b, i] = 0
                k[b, i] = 0
                continue
            if rope:
                cos, sin = (t[p].double() for t in s.rope)
                q[b, i], k[b, i] = (rotated(x[b, i], cos, sin, interleaved) for x in (q, k))
            where = place(s, b, p)
            if where is None:
                continue
            for target, x in zip(pages, (k[b, i], s.v[b, i].double())):
                target[where[0], :, where[1]] = four_bit(x) if s.bits == 4 else x
    return q, k, pages[0], pages[1]


def gather(s):
    out = [torch.zeros(s.batch, s.tokens, *(x.shape[1], x.shape[3]), dtype=torch.float64)
           for x in s.held]
    for b in range(s.batch):
        for i in range(s.tokens):
            p = live_position(s, b, i)
            where = None if p is None else place(s, b, p)
            if where is not None:
                for x, held in zip(out, s.held):
                    x[b, i] = held[where[0], :, where[1]].double()
    return out


def attention(s, scale):
    """out, lse, and the bounds of their errors without the output's own rounding. With P|V| the
    attention of |v|, and S the largest scale |q| |k| of a row's keys: a score in fp32 is off by at
    most (D + 2) 2^-24 S (D products and sums), so a probability by twice that, relatively;
    holding it in two bf16 parts adds 2^-16, its exponential and the running sums of up to 2^17
    keys in blocks 2^-17: an output by the sum of these times P|V|, an LSE by the score's error
    plus 2^-20 of itself. A probability below fp32's normal range, 2^-126, may be taken as 0: an
    output by another 2^-126 of the sum of |v|."""
    batch, tokens, heads, dim = s.q.shape
    out = torch.zeros(s.q.shape, dtype=torch.float64)
    lse = torch.full((batch, tokens, heads), -math.inf, dtype=torch.float64)
    out_off, lse_off = torch.zeros_like(out), torch.zeros_like(lse)
    group = heads // s.held[0].shape[1]
    for b in range(batch):
        for i in range(tokens):
            p = live_position(s, b, i)
            if p is None:
                continue
            at = torch.arange(p + 1)
            ids = s.table[b].long()[at // s.page]
            ok = (ids >= 0) & (ids < s.pages)
            if not ok.any():
                continue
            k, v = (x[ids[ok], :, (at % s.page)[ok]].double().repeat_interleave(group, 1)
                    for x in s.held)
            q = s.q[b, i].double()
            logits = (k * q).sum(-1) * scale
            weights = torch.softmax(logits, 0)[..., None]
            lse[b, i] = torch.logsumexp(logits, 0)
            out[b, i] = (weights * v).sum(0)
            off = (k.abs() * q.abs()).sum(-1).amax(0) * abs(scale) * (dim + 2) * 2.0 ** -24
            out_off[b, i] = (weights * v.abs()).sum(0) * (2 * off[:, None] + 2.0 ** -16 + 2.0 ** -17) \
                + 2.0 ** -126 * v.abs().sum(0)
            lse_off[b, i] = off + 2.0 ** -20 * (1 + lse[b, i].abs())
    return out, lse, out_off, lse_off
