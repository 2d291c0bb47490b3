"""Drafted trees and evictions of the paged cache in 64 bits on the CPU."""

from __future__ import annotations

import math

import torch

import paged_reference as ref


def random_parents(seed, batch, tokens):
    gen = torch.Generator().manual_seed(seed)
    up = torch.rand(batch, tokens, generator=gen) ** 0.6 * torch.arange(tokens)
    parents = up.floor().long().minimum((torch.arange(tokens) - 1).clamp(min=0)).int()
    parents[:, 0] = -1
    return parents


def lineage(parents):
    """[B, T] -> bool [B, T, T] (j is i or an ancestor of it), depths."""
    batch, tokens = parents.shape
    seen = torch.zeros(batch, tokens, tokens, dtype=torch.bool)
    depth = torch.zeros(batch, tokens, dtype=torch.int32)
    for b in range(batch):
        for i in range(tokens):
            seen[b, i, i] = True
            p = int(parents[b, i])
            if 0 <= p < i:
                seen[b, i] |= seen[b, p]
                depth[b, i] = depth[b, p] + 1
    return seen, depth


def words(seen):
    """bool [B, T, J] -> int64 [B, T, ceil(J / 64)]."""
    out = torch.zeros(*seen.shape[:2], -(-seen.shape[2] // 64), dtype=torch.int64)
    for j in range(seen.shape[2]):
        bit = 1 << (j % 64)
        out[..., j // 64] |= torch.where(seen[..., j], bit - (1 << 64) if j % 64 == 63 else bit, 0)
    return out


def live_tokens(s, b):
    return sum(ref.live_position(s, b, i) is not None for i in range(s.tokens))


def tree_attention(s, seen, scale):
    """out, lse, and the bounds of their errors without the output's own rounding; seen: [B, T, T].

    With S the largest scale |q| |k| of a row's keys a score in fp32 is off by (D + 2) 2^-24 S, a
    probability by twice that, relatively. Its exponential adds 2^-22, the sums of n keys, 32 at a
    time in a tree, then one after the other and over at most 1024 workgroups,
    (n / 32 + 1024 / 32 + 16) 2^-24; two bf16 parts of it 2^-18 and the products' sum of a lane's
    16 keys at a time another (n / 16 + 64) 2^-24 of the sum of p |v|. A probability below 2^-126 may
    be 0."""
    batch, tokens, heads, dim = s.q.shape
    out = torch.zeros(s.q.shape, dtype=torch.float64)
    lse = torch.full((batch, tokens, heads), -math.inf, dtype=torch.float64)
    out_off, lse_off = torch.zeros_like(out), torch.zeros_like(lse)
    group = heads // s.held[0].shape[1]
    for b in range(batch):
        live = live_tokens(s, b)
        if live == 0:
            continue
        start = int(s.starts[b])
        at = torch.arange(start + live)
        ids = s.table[b].long()[at // s.page]
        placed = (ids >= 0) & (ids < s.pages)
        rows = [x[ids.clamp(0, s.pages - 1), :, at % s.page].double().repeat_interleave(group, 1)
                for x in s.held]
        for i in range(live):
            ok = placed & torch.cat((torch.ones(start, dtype=torch.bool), seen[b, i, :live]))
            if not ok.any():
                continue
            k, v = (x[ok] for x in rows)
            q = s.q[b, i].double()
            logits = (k * q).sum(-1) * scale
            weights = torch.softmax(logits, 0)[..., None]
            lse[b, i] = torch.logsumexp(logits, 0)
            out[b, i] = (weights * v).sum(0)
            off = (k.abs() * q.abs()).sum(-1).amax(0) * abs(scale) * (dim + 2) * 2.0 ** -24
            n = start + live
            sums = (n / 32 + 48) * 2.0 ** -24 + 2.0 ** -22
            parts = 2.0 ** -18 + (n / 16 + 64) * 2.0 ** -24
            out_off[b, i] = (weights * v.abs()).sum(0) * (2 * off[:, None] + sums + parts) \
                + 2.0 ** -126 * v.abs().sum(0)
            lse_off[b, i] = off + sums + 2.0 ** -22 * (1 + lse[b, i].abs())
    return out, lse, out_off, lse_off


def accept(parents, drafts, targets, live):
    """The accepted nodes of one tree."""
    path = [0] if live else []
    while path:
        after = [i for i in range(path[-1] + 1, live)
                 if parents[i] == path[-1] and drafts[i] == targets[path[-1]]]
        if not after:
            break
        path.append(after[0])
    return path


def move(s, pages, b, pairs):
    """Rows of all heads from position to position, in order, where both have a place."""
    for to, of in pairs:
        target, source = ref.place(s, b, to), ref.place(s, b, of)
        if target and source:
            for x in pages:
                x[target[0], :, target[1]] = x[source[0], :, source[1]].clone()


def gathered(s, lse, scale):
    """Sum of probabilities per key, float64 [B, Hkv, reach], and the bound of its error: a score is
    off by (D + 2) 2^-24 of scale |q| |k| and 2^-22 of itself and the LSE in base 2, which the
    exponential takes as a relative error, and adds 2^-22; the sums of c columns, one after the
    other, c 2^-24."""
    batch, tokens, heads, dim = s.q.shape
    kv = s.held[0].shape[1]
    group = heads // kv
    reach = s.table.shape[1] * s.page
    total = torch.zeros(batch, kv, reach, dtype=torch.float64)
    off = torch.zeros_like(total)
    for b in range(batch):
        for i in range(tokens):
            p = ref.live_position(s, b, i)
            if p is None:
                continue
            at = torch.arange(p + 1)
            ids = s.table[b].long()[at // s.page]
            placed = (ids >= 0) & (ids < s.pages)
            k = s.held[0][ids.clamp(0, s.pages - 1), :, at % s.page].double()
            for h in range(heads):
                row = float(lse[b, i, h])
                if row == -math.inf:
                    continue
                q, mine = s.q[b, i, h].double(), k[:, h // group]
                w = torch.exp((mine @ q) * scale - row) * placed
                w = torch.where(placed, w, 0)
                wrong = (mine.abs() @ q.abs()) * abs(scale) * (dim + 2) * 2.0 ** -24 \
                    + 2.0 ** -22 * (2 + abs(row) + 16) + tokens * group * 2.0 ** -24
                total[b, h // group, :p + 1] += w
                off[b, h // group, :p + 1] += torch.where(placed, w * wrong, 0)
    return total, off


def evict(s, lengths, weights, budget, positions, seen, recent, sinks):
    """(lengths, weights, positions, key pages, value pages); weights float32 [B, Hkv, slots]."""
    batch, kv, slots = weights.shape
    reach = s.table.shape[1] * s.page
    lengths_out, pages = lengths.clone(), [x.clone() for x in s.held]
    weights_out, positions_out = torch.zeros_like(weights), torch.full_like(weights, -1).int()
    for b in range(batch):
        n = int(lengths[b])
        text = n if seen is None else int(seen[b])
        keep = max(0, min(n, slots))
        weights_out[b, :, :keep] = weights[b, :, :keep]
        if positions is not None:
            positions_out[b, :, :keep] = positions[b, :, :keep]
        if n <= budget or n > reach or any(ref.place(s, b, p) is None for p in range(0, n, s.page)):
            continue
        lengths_out[b] = budget
        for h in range(kv):
            def position(p):
                told = -1 if positions is None else int(positions[b, h, p])
                return told if told >= 0 else text - n + p

            def order(p):
                w = float(weights[b, h, p])
                safe = position(p) < sinks or position(p) >= text - recent
                return (not safe, math.isnan(w), -w if w == w else 0.0, p)

            stay = set(sorted(range(n), key=order)[:budget])
            places = list(range(budget))
            free = [p for p in places if p not in stay]
            for to, of in zip(free, sorted(p for p in stay if p >= budget)):
                places[to] = of
                target, source = ref.place(s, b, to), ref.place(s, b, of)
                for x, y in zip(pages, s.held):
                    x[target[0], h, target[1]] = y[source[0], h, source[1]]
            weights_out[b, h] = 0
            positions_out[b, h] = -1
            weights_out[b, h, :budget] = weights[b, h, places]
            positions_out[b, h, :budget] = torch.tensor([position(p) for p in places])
    return lengths_out, weights_out, positions_out, pages[0], pages[1]
