"""Cases of drafted trees and of eviction in the paged KV cache: attention of a tree of drafted
tokens, acceptance of the drafts that the model agrees with, the attention weight that cached
tokens gather, and eviction of those that gathered least.

Pages are ``[pages, Hkv, page_size, D]`` in bfloat16, or in 4 bits: E2M1 values (0, 0.5, 1,
1.5, 2, 3, 4, 6 and a sign), two per byte with the even dim in the low half, and one
power-of-two scale (E8M0, bias 127) per token, head and 32 dims.

``run`` computes a case in plain torch operations, or, with ``own`` set, through
``exp3_amd.paged``.
"""

from __future__ import annotations

import math

import numpy
import torch

own = False

GROUP = 32                      # dims per scale of a 4-bit page
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# (query heads, KV heads, head dim): Qwen2.5-7B, Llama-like 4:1, Qwen2.5-1.5B, no GQA, and the
# Qwen3.5 full-attention layers
LAYOUTS = ((28, 4, 128), (32, 8, 128), (12, 2, 128), (8, 8, 128), (16, 4, 256))


def _case(op, keys, layout=LAYOUTS[0], batch=1, tokens=1, bits=16, page=16, ragged=False, **more):
    """keys: those of the longest sequence, its new tokens among them; tokens: new ones per
    sequence. Ragged batches have shorter sequences and, from four sequences on, a free slot."""
    return dict(op=op, keys=keys, batch=batch, tokens=tokens, bits=bits, page=page, ragged=ragged,
                q_heads=layout[0], kv_heads=layout[1], dim=layout[2], **more)


def listed():
    return [
        # a small tree behind a short prompt: launches and latency
        _case("tree", 1106, tokens=16, name="tree_t16_1106"),
        # a batch of long conversations of unlike lengths
        _case("tree", 16000, LAYOUTS[1], batch=8, tokens=32, page=128, ragged=True,
              name="tree_b8_t32_16000"),
        # large trees of a serving batch in 4 bits
        _case("tree", 8192, batch=16, tokens=61, bits=4, page=16, ragged=True,
              name="tree_4bit_b16_t61_8192"),
        # head dim 256 in 4 bits
        _case("tree", 12001, LAYOUTS[4], batch=4, tokens=26, bits=4, page=64, ragged=True,
              name="tree_4bit_d256_t26"),
        # the drafts of one chat, all layers of a model
        _case("accept", 1106, tokens=16, layers=28, name="accept_t16_28_layers"),
        # a serving batch with large trees
        _case("accept", 300, LAYOUTS[1], batch=64, tokens=61, page=32, ragged=True, layers=12,
              name="accept_b64_t61_12_layers"),
        # a decode step of a serving batch in 4 bits
        _case("weights", 8192, LAYOUTS[1], batch=64, bits=4, page=16, ragged=True,
              name="weights_4bit_b64_8192"),
        # the last 64 tokens of a 32K prompt judge the others
        _case("weights", 32640, tokens=64, page=128, name="weights_t64_32640"),
        # a chunk of a prompt behind a cached prefix
        _case("weights", 16000, tokens=2000, page=64, name="weights_chunk_2000_16000"),
        # a few tokens over the budget: what every so many steps costs
        _case("evict", 2112, LAYOUTS[1], batch=64, page=32, budget=2048, recent=256, sinks=4,
              again=True, name="evict_b64_2112_to_2048"),
        # a prompt cut down to an eighth
        _case("evict", 32640, page=128, budget=4096, recent=64, sinks=4, again=False,
              name="evict_32640_to_4096"),
        # conversations of unlike lengths in 4 bits, some within the budget already
        _case("evict", 9001, LAYOUTS[4], batch=8, bits=4, page=64, ragged=True, budget=3001,
              recent=100, sinks=0, again=True, name="evict_4bit_b8_9001_to_3001"),
    ]


def _length(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(("tree", "tree", "tree", "accept", "weights", "weights", "evict", "evict"))
    layout = rng.choice(LAYOUTS)
    bits, page = rng.choice((16, 4)), rng.choice((16, 32, 64, 128))
    ragged = rng.random() < 0.5
    row = layout[1] * layout[2]                    # elements of one token's keys
    if op == "tree":
        batch, tokens = rng.choice((1, 1, 2, 4, 9, 16)), _length(rng, 2, 130)
        pairs = 100_000_000 // (batch * tokens * layout[0])
        most = min(40000, pairs, (100_000_000 if bits == 16 else 200_000_000) // (row * batch))
        return _case(op, _length(rng, tokens, max(tokens, most)), layout, batch, tokens, bits, page,
                     ragged)
    if op == "accept":
        batch, tokens, layers = rng.choice((1, 2, 5, 16, 64)), _length(rng, 2, 64), rng.randint(1, 28)
        most = 100_000_000 // (row * batch * layers)
        return _case(op, _length(rng, tokens, max(tokens + 1, min(4000, most))), layout, batch,
                     tokens, 16, page, ragged, layers=layers)
    if op == "weights":
        batch = rng.choice((1, 1, 2, 3, 8, 24, 64))
        tokens = rng.choice((1, 1, 1, 2, 5, 16, 33, 64, 301, 1000))
        pairs = 400_000_000 // (batch * tokens * layout[0])
        most = min(100000, pairs, (130_000_000 if bits == 16 else 300_000_000) // (row * batch))
        return _case(op, _length(rng, tokens, max(tokens, most)), layout, batch, tokens, bits, page,
                     ragged)
    batch = rng.choice((1, 1, 2, 7, 24, 64))
    keys = _length(rng, 40, min(60000, 100_000_000 // (row * batch)))
    budget = max(1, int(keys * rng.choice((0.1, 0.25, 0.5, 0.9, 0.98, 1.0))))
    return _case(op, keys, layout, batch, 1, bits, page, ragged, budget=budget,
                 recent=rng.randint(0, budget // 2), sinks=rng.choice((0, 0, 1, 4)) % (budget // 2 + 1),
                 again=rng.random() < 0.5)


def _plan(case):
    """(tokens held before, new tokens) per sequence; -1 held: a free slot."""
    held, new = [], []
    for b in range(case["batch"]):
        share = 1.0 if not case["ragged"] else 1.0 - 0.9 * (b * 0.6180339887 % 1.0)
        count = max(1, int(case["tokens"] * share))
        keys = max(count, int(case["keys"] * share))
        free = case["ragged"] and b % 16 == 3
        held.append(-1 if free else keys - count)
        new.append(0 if free else count)
    return held, new


# ------------------------------------------------------------------- inputs

def _to_4bit(x):
    """[..., D] -> packed E2M1 values [..., D / 2] and E8M0 scales [..., D / 32]: the scale that
    puts the largest of its 32 values into [3.5, 7), values to the nearest code."""
    x = x.unflatten(-1, (-1, GROUP))
    mantissa, exponent = torch.frexp(x.abs().amax(-1))
    scale = (exponent + (mantissa >= 0.875) + 124).clamp(2, 252)
    y = torch.ldexp(x.abs(), (127 - scale)[..., None])
    code = torch.bucketize(y, torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), device=x.device))
    code = code.to(torch.uint8) | (x < 0).to(torch.uint8) << 3
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] | code[..., 1] << 4, scale.to(torch.uint8)


def _tree(batch, tokens, gen, device):
    """Parents of random trees, breadth first: node i > 0 hangs on one of the nodes before it, most
    often on one some way back."""
    back = torch.rand(batch, tokens, generator=gen, device=device) ** 0.7
    node = torch.arange(tokens, device=device)
    parents = (back * node).floor().long().clamp(max=tokens).minimum((node - 1).clamp(min=0))
    parents[:, 0] = -1
    return parents


def _ancestors(parents):
    """[B, T, T]: whether node j is node i or one of its ancestors."""
    batch, tokens = parents.shape
    node = torch.arange(tokens, device=parents.device)
    seen = (parents[..., None] == node) | (node[:, None] == node)
    for _ in range(tokens.bit_length()):
        seen = (seen.float() @ seen.float()) > 0
    return seen


def _words(seen):
    """[B, T, J] truth values -> int64 [B, T, ceil(J / 64)], bit j % 64 of word j // 64."""
    pad = -seen.shape[-1] % 64
    bits = torch.nn.functional.pad(seen, (0, pad)).unflatten(-1, (-1, 64)).long()
    return (bits << torch.arange(64, device=seen.device)).sum(-1)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device).manual_seed(seed)
    op, batch, tokens, page = case["op"], case["batch"], case["tokens"], case["page"]
    heads, kv, dim = case["q_heads"], case["kv_heads"], case["dim"]
    held, new = _plan(case)
    width = -(-case["keys"] // page)
    reach, pages = width * page, batch * width + 3

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    # page ids as a server's free list leaves them: in no order
    table = torch.randperm(pages, generator=gen, device=device)[:batch * width]
    state = dict(case=case, scale=dim ** -0.5,
                 table=table.view(batch, width).to(torch.int32),
                 starts=torch.tensor(held, dtype=torch.int32, device=device),
                 counts=torch.tensor(new, dtype=torch.int32, device=device)
                 if case["ragged"] else None)
    # keys with channels of unlike size, as projections with biases leave them
    gain = torch.exp(0.5 * normal(kv, 1, dim))
    layers = case.get("layers", 0)
    total = pages * max(layers, 1)
    for name, size in (("key", gain), ("value", 1.0)):
        held_pages, scales = [], []
        for part in torch.arange(total, device=device).split(max(1, (1 << 27) // (kv * page * dim))):
            x = (normal(part.numel(), kv, page, dim) * size).to(torch.bfloat16)
            if case["bits"] == 4:
                x, scale = _to_4bit(x.float())
                scales.append(scale)
            held_pages.append(x)
        held_pages = torch.cat(held_pages)
        state[name + "_pages"] = held_pages.unflatten(0, (layers, pages)) if layers else held_pages
        state[name + "_scales"] = torch.cat(scales) if scales else None
    sharp = torch.linspace(0.3, 2.0, heads, device=device)[:, None]
    if op in ("tree", "accept"):
        parents = _tree(batch, tokens, gen, device)
        state |= dict(parents=parents.to(torch.int32), masks=_words(_ancestors(parents)))
    if op == "tree":
        state["q"] = (normal(batch, tokens, heads, dim) * sharp).to(torch.bfloat16)
    elif op == "accept":
        # a token of a small vocabulary per node, so that some drafts are what the model chose
        state["drafts"] = torch.randint(0, 3, (batch, tokens), generator=gen, device=device)
        state["targets"] = torch.randint(0, 3, (batch, tokens), generator=gen, device=device)
    elif op == "weights":
        state["q"] = (normal(batch, tokens, heads, dim) * sharp).to(torch.bfloat16)
        state["lse"] = _row_sums(state)
        # what some decode steps have left, or a prompt's tokens before anything looked at them
        state["weights"] = torch.rand(batch, kv, reach, generator=gen, device=device) * \
            (0.02 if tokens < 16 else 0.0) * \
            (torch.arange(reach, device=device) < state["starts"][:, None, None])
    elif op == "evict":
        state |= _ledger(case, state, reach, gen, device)
    return state


def _ledger(case, state, reach, gen, device):
    """Lengths, gathered weights (a fifth of them 0: tokens that nothing looked at) and, where an
    eviction came before, the positions that it left: all but the last few tokens have moved."""
    batch, kv = case["batch"], case["kv_heads"]
    slot = torch.arange(reach, device=device)
    lengths = torch.where(state["starts"] < 0, -1, state["starts"] + 1).to(torch.int32)
    weights = torch.exp(2 * torch.randn(batch, kv, reach, generator=gen, device=device))
    weights *= torch.rand(batch, kv, reach, generator=gen, device=device) > 0.2
    weights *= slot < lengths[:, None, None]
    out = dict(lengths=lengths, weights=weights, positions=None, seen=None)
    if case["again"]:
        text = lengths.clamp(min=0).long() * 3
        recorded = (lengths.long() - lengths.long() // 16).clamp(min=0)[:, None, None]
        # distinct positions in no order, below those of the tokens that came after
        mixed = torch.rand(batch, kv, reach, generator=gen, device=device)
        mixed = mixed.masked_fill(slot >= recorded, 2.0).argsort(-1).argsort(-1) * 2
        out["positions"] = torch.where(slot < recorded, mixed, -1).to(torch.int32)
        out["seen"] = text.to(torch.int32)
    return out


# -------------------------------------------------------------- plain forms

def _from_4bit(packed, scale):
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    value = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=packed.device)[code.long()]
    size = torch.ldexp(torch.ones((), device=packed.device), scale.int() - 127)
    return (value.unflatten(-1, (-1, GROUP)) * size[..., None]).flatten(-2)


def _places(state):
    """[B, T] positions of the new tokens and whether each is a token."""
    case, starts = state["case"], state["starts"].long()
    step = torch.arange(case["tokens"], device=starts.device)
    count = case["tokens"] if state["counts"] is None else state["counts"].long()[:, None]
    where = starts[:, None] + step
    return where, (starts[:, None] >= 0) & (step < count)


def _held(state, name):
    """[B, Hkv, reach, D] in fp32: the keys or values that the page table names."""
    case, at = state["case"], state["table"].long()
    x = state[name + "_pages"][at]
    if case["bits"] == 4:
        x = _from_4bit(x, state[name + "_scales"][at])
    return x.transpose(1, 2).reshape(case["batch"], case["kv_heads"], -1, case["dim"]).float()


def _logits(state, seen):
    """[B, Hkv, T, group, reach] scores, -inf where a token does not see a key."""
    case, q = state["case"], state["q"]
    batch, tokens, heads, dim = q.shape
    kv = case["kv_heads"]
    rows = q.float().view(batch, tokens, kv, heads // kv, dim).permute(0, 2, 1, 3, 4)
    logits = rows.reshape(batch, kv, -1, dim) @ _held(state, "key").transpose(2, 3)
    logits = (logits * state["scale"]).view(batch, kv, tokens, heads // kv, -1)
    return logits.masked_fill_(~seen[:, None, :, None], -math.inf)


def _causal(state):
    where, live = _places(state)
    reach = state["table"].shape[1] * state["case"]["page"]
    return live[..., None] & (torch.arange(reach, device=where.device) <= where[..., None])


def _row_sums(state):
    """Natural-log LSE of the new tokens' rows, [B, T, Hq]."""
    lse = torch.logsumexp(_logits(state, _causal(state)), -1)
    return lse.permute(0, 2, 1, 3).reshape(state["q"].shape[:3])


def _plain_tree(state):
    case, q, masks = state["case"], state["q"], state["masks"]
    batch, tokens, heads, dim = q.shape
    kv = case["kv_heads"]
    _, live = _places(state)
    key = torch.arange(state["table"].shape[1] * case["page"], device=q.device)
    draft = key - state["starts"].long()[:, None]                 # [B, reach]
    bit = draft.clamp(0, tokens - 1)[:, None].expand(-1, tokens, -1)
    drafted = (masks.gather(2, bit // 64) >> (bit % 64) & 1).bool()
    drafted &= ((draft < tokens) & live.gather(1, draft.clamp(0, tokens - 1)))[:, None]
    logits = _logits(state, live[..., None] & ((draft < 0)[:, None] | drafted))
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(torch.isinf(top), 0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1, total)
    out = (p.view(batch, kv, -1, key.numel()) @ _held(state, "value")).view(batch, kv, tokens, -1, dim)
    lse = (total.log() + top)[..., 0]
    return {"out": out.permute(0, 2, 1, 3, 4).reshape(q.shape).to(torch.bfloat16),
            "lse": lse.permute(0, 2, 1, 3).reshape(batch, tokens, heads)}


def _plain_accept(state):
    case, parents, masks = state["case"], state["parents"].long(), state["masks"]
    batch, tokens = parents.shape
    page = case["page"]
    where, live = _places(state)
    node = torch.arange(tokens, device=parents.device)
    drafts, targets = state["drafts"], state["targets"]
    match = (drafts == targets.gather(1, parents.clamp(min=0))) & (parents >= 0) & live
    sooner = (parents[:, :, None] == parents[:, None]) & match[:, None] & (node < node[:, None])
    good = match & ~sooner.any(-1)
    good[:, 0] = live[:, 0]
    seen = (masks[..., node // 64] >> (node % 64) & 1).bool()     # [B, T, T]
    taken = ~(seen & ~good[:, None]).any(-1)
    count = taken.sum(-1)
    path = torch.where(taken, node, tokens).sort(-1).values
    last = path.gather(1, (count - 1).clamp(min=0)[:, None]).clamp(max=tokens - 1)
    following = torch.where(count > 0, targets.gather(1, last)[:, 0], -1)
    b, step = (node < count[:, None]).nonzero(as_tuple=True)
    start, table = state["starts"].long()[b], state["table"].long()
    source, target = start + path[b, step], start + step
    for name in ("key_pages", "value_pages"):
        held = state[name].transpose(2, 3)                        # [layers, pages, page, Hkv, D]
        held[:, table[b, target // page], target % page] = \
            held[:, table[b, source // page], source % page]
    return {"accepted": count.int(), "path": torch.where(path < tokens, path, -1).int(),
            "following": following, "key_pages": state["key_pages"],
            "value_pages": state["value_pages"]}


def _plain_weights(state):
    case = state["case"]
    batch, tokens, heads, _ = state["q"].shape
    kv = case["kv_heads"]
    lse = state["lse"].view(batch, tokens, kv, heads // kv).permute(0, 2, 1, 3)
    logits = _logits(state, _causal(state))
    p = torch.exp(logits.sub_(torch.where(torch.isinf(lse), 0, lse)[..., None]))
    state["weights"] += p.sum((2, 3))
    return {"weights": state["weights"]}


def _plain_evict(state):
    case, weights, table = state["case"], state["weights"], state["table"].long()
    budget, page = case["budget"], case["page"]
    reach = weights.shape[2]
    slot = torch.arange(reach, device=weights.device)
    lengths = state["lengths"].long()[:, None, None]
    seen = lengths if state["seen"] is None else state["seen"].long()[:, None, None]
    told = torch.full_like(weights, -1).long() if state["positions"] is None \
        else state["positions"].long()
    positions = torch.where(told < 0, seen - lengths + slot, told)
    order = weights.masked_fill((positions < case["sinks"]) | (positions >= seen - case["recent"]),
                                math.inf).masked_fill(slot >= lengths, -math.inf)
    rank = torch.sort(order, stable=True, dim=-1, descending=True).indices.argsort(-1)
    kept = (rank < budget) & (slot < lengths)
    cut = lengths > budget
    target = (cut & ~kept & (slot < budget)).nonzero(as_tuple=True)
    source = (cut & kept & (slot >= budget)).nonzero(as_tuple=True)
    left = torch.where(cut, budget, lengths)
    new_weights = torch.where(slot < left, weights, 0)
    new_positions = torch.where(slot < left, torch.where(cut, positions, told), -1)
    new_weights[target], new_positions[target] = weights[source], positions[source]
    to, of = ((table[b, s // page], h, s % page) for b, h, s in (target, source))
    state["key_pages"][to] = state["key_pages"][of]
    state["value_pages"][to] = state["value_pages"][of]
    out = {"lengths": left[:, 0, 0].int(), "weights": new_weights, "positions": new_positions.int()}
    if case["bits"] == 16:
        return out | {"key_pages": state["key_pages"], "value_pages": state["value_pages"]}
    state["key_scales"][to] = state["key_scales"][of]
    state["value_scales"][to] = state["value_scales"][of]
    here = (slot[:budget] < left[:, 0])[:, :, None, None]
    at = table[:, slot[:budget] // page]
    keys, values = (_from_4bit(state[name + "_pages"][at, :, slot[:budget] % page],
                               state[name + "_scales"][at, :, slot[:budget] % page])
                    .to(torch.bfloat16).masked_fill(~here, 0) for name in ("key", "value"))
    return out | {"keys": keys, "values": values}


# ---------------------------------------------------------------------- run

def _own(state):
    from exp3_amd import paged

    case = state["case"]
    place = (state["table"], state["starts"])
    if case["op"] == "accept":
        caches = [paged.PagedCache(k, v) for k, v in zip(state["key_pages"], state["value_pages"])]
        accepted, path, following = paged.accept_drafts(
            caches, *place, state["parents"], state["drafts"], state["targets"], state["counts"])
        return {"accepted": accepted, "path": path, "following": following,
                "key_pages": state["key_pages"], "value_pages": state["value_pages"]}
    cache = paged.PagedCache(state["key_pages"], state["value_pages"], state["key_scales"],
                             state["value_scales"])
    if case["op"] == "tree":
        out, lse = paged.tree_attention(state["q"], cache, *place, state["masks"], state["scale"],
                                        state["counts"], return_lse=True)
        return {"out": out, "lse": lse}
    if case["op"] == "weights":
        paged.accumulate_weights(state["weights"], state["q"], state["lse"], cache, *place,
                                 state["scale"], state["counts"])
        return {"weights": state["weights"]}
    lengths, weights, positions = paged.evict_tokens(
        cache, state["table"], state["lengths"], state["weights"], case["budget"],
        state["positions"], state["seen"], case["recent"], case["sinks"])
    out = {"lengths": lengths, "weights": weights, "positions": positions}
    if case["bits"] == 16:
        return out | {"key_pages": cache.key_pages, "value_pages": cache.value_pages}
    first = torch.where(lengths < 0, -1, 0).int()
    keys, values = paged.gather_tokens(cache, state["table"], first, case["budget"], lengths)
    return out | {"keys": keys, "values": values}


def run(state):
    if own:
        return _own(state)
    return {"tree": _plain_tree, "accept": _plain_accept, "weights": _plain_weights,
            "evict": _plain_evict}[state["case"]["op"]](state)


# --------------------------------------------------------------------- work

def work(case):
    held, new = _plan(case)
    batch, heads, kv, dim = case["batch"], case["q_heads"], case["kv_heads"], case["dim"]
    row = dim * 2 if case["bits"] == 16 else dim // 2 + dim // GROUP
    wide = batch * case["tokens"] * heads * dim * 2       # bf16 rows of the queries, padding too
    reach = -(-case["keys"] // case["page"]) * case["page"]
    if case["op"] == "accept":
        # some two of the accepted tokens are not in their place yet
        moved = 2 * sum(n > 2 for n in new) * case["layers"]
        return {"bytes": 4 * kv * row * moved + batch * case["tokens"] * (4 + 8 + 8 + 4) + batch * 16,
                "flops": 0}
    if case["op"] == "evict":
        lengths = [h + n for h, n in zip(held, new) if h >= 0]
        budget = case["budget"]
        # of the tokens behind the budget's end the share that stays is the one of all tokens
        moved = sum((n - budget) * budget // n for n in lengths if n > budget)
        entry = 8 if case["again"] else 4
        size = 4 * row * kv * moved + kv * (entry * sum(lengths) + 8 * batch * reach)
        if case["bits"] == 4:       # read back as values
            size += 2 * kv * (row * sum(min(n, budget) for n in lengths) + batch * budget * dim * 2)
        return {"bytes": size, "flops": 0}
    keys = sum(h + n for h, n in zip(held, new) if h >= 0)
    if case["op"] == "tree":        # a node sees the cache, itself and a few ancestors
        pairs = sum(n * (h + 1 + n.bit_length() // 2) for h, n in zip(held, new) if h >= 0)
        return {"bytes": 2 * kv * row * keys + 2 * wide + 2 * wide // dim + 8 * batch * case["tokens"],
                "flops": 4 * heads * dim * pairs}
    pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new) if h >= 0)
    return {"bytes": kv * (row + 8) * keys + wide + 2 * wide // dim, "flops": 2 * heads * dim * pairs}


# -------------------------------------------------------------------- exact

def _rows(state, name, b, count):
    """[count, Hkv, D] in float64 of sequence b's first tokens."""
    page = state["case"]["page"]
    at = torch.arange(count, device=state["table"].device)
    ids = state["table"][b].long()[torch.div(at, page, rounding_mode="floor")]
    rows = state[name + "_pages"][ids, :, at % page]
    if state["case"]["bits"] == 16:
        return rows.double()
    values = torch.tensor([(-1.0) ** (c >> 3) * E2M1[c & 7] for c in range(16)],
                          dtype=torch.float64, device=rows.device)
    pairs = torch.stack((values[(rows % 16).long()], values[(rows // 16).long()]), -1)
    exponent = state[name + "_scales"][ids, :, at % page].double() - 127
    return pairs.reshape(*rows.shape[:2], -1, GROUP).mul(2.0 ** exponent[..., None]).flatten(2)


def _lineage(parents):
    """Every node's ancestors and itself, walked upwards."""
    found = []
    for i in range(len(parents)):
        line = [i]
        while parents[line[-1]] >= 0:
            line.append(parents[line[-1]])
        found.append(sorted(line))
    return found


def exact(case, seed):
    state = prepare(case, seed)
    return {"tree": _exact_tree, "accept": _exact_accept, "weights": _exact_weights,
            "evict": _exact_evict}[case["op"]](case, state, *_plan(case))


def _exact_tree(case, state, held, new):
    batch, tokens, heads, group = case["batch"], case["tokens"], case["q_heads"], \
        case["q_heads"] // case["kv_heads"]
    device = state["table"].device
    out = torch.zeros(batch, tokens, heads, case["dim"], dtype=torch.float64, device=device)
    lse = torch.full((batch, tokens, heads), -math.inf, dtype=torch.float64, device=device)
    parents = state["parents"].tolist()
    for b in range(batch):
        if held[b] < 0:
            continue
        k, v = (_rows(state, name, b, held[b] + new[b]) for name in ("key", "value"))
        hidden = torch.ones(new[b], held[b] + new[b], dtype=torch.bool, device=device)
        hidden[:, :held[b]] = False
        for i, line in enumerate(_lineage(parents[b])[:new[b]]):
            hidden[i, [held[b] + j for j in line]] = False
        for h in range(heads):
            logits = state["q"][b, :new[b], h].double() @ k[:, h // group].T * state["scale"]
            logits[hidden] = -math.inf
            lse[b, :new[b], h] = torch.logsumexp(logits, 1)
            out[b, :new[b], h] = torch.softmax(logits, 1) @ v[:, h // group]
    return {"out": out, "lse": lse}


def _exact_accept(case, state, held, new):
    page = case["page"]
    pages = [state[name].double() for name in ("key_pages", "value_pages")]
    parents, drafts, targets = (state[name].tolist() for name in ("parents", "drafts", "targets"))
    table = state["table"].tolist()
    for b in range(case["batch"]):
        path = [0] if new[b] else []
        while path:
            after = [i for i in range(new[b]) if parents[b][i] == path[-1]
                     and drafts[b][i] == targets[b][path[-1]]]
            if not after:
                break
            path.append(after[0])
        for j, i in enumerate(path):
            (to, at), (of, was) = (divmod(held[b] + x, page) for x in (j, i))
            for x in pages:
                x[:, table[b][to], :, at] = x[:, table[b][of], :, was].clone()
    return {"accepted": None, "path": None, "following": None, "key_pages": pages[0],
            "value_pages": pages[1]}


def _exact_weights(case, state, held, new):
    group = case["q_heads"] // case["kv_heads"]
    total = state["weights"].double()
    for b in range(case["batch"]):
        if held[b] < 0:
            continue
        k = _rows(state, "key", b, held[b] + new[b])
        later = torch.arange(held[b] + new[b], device=k.device) > \
            held[b] + torch.arange(new[b], device=k.device)[:, None]
        for h in range(case["q_heads"]):
            logits = state["q"][b, :new[b], h].double() @ k[:, h // group].T * state["scale"]
            p = torch.exp(logits - state["lse"][b, :new[b], h, None].double())
            total[b, h // group, :held[b] + new[b]] += p.masked_fill_(later, 0).sum(0)
    return {"weights": total}


def _exact_evict(case, state, held, new):
    budget, page, kv = case["budget"], case["page"], case["kv_heads"]
    pages = [state[name + "_pages"] for name in ("key", "value")]
    weights, table = state["weights"].double(), state["table"].long()
    moves = []
    for b in range(case["batch"]):
        n = int(state["lengths"][b])
        if n <= budget:
            continue
        seen = n if state["seen"] is None else int(state["seen"][b])
        for h in range(kv):
            position = torch.arange(seen - n, seen, device=weights.device)
            if state["positions"] is not None:
                told = state["positions"][b, h, :n].long()
                position = torch.where(told >= 0, told, position)
            safe = (position < case["sinks"]) | (position >= seen - case["recent"])
            # the last key counts first
            order = numpy.lexsort((range(n), -weights[b, h, :n].cpu().numpy(), ~safe.cpu().numpy()))
            stay = numpy.zeros(n, dtype=bool)
            stay[order[:budget]] = True
            free, far = numpy.flatnonzero(~stay[:budget]), budget + numpy.flatnonzero(stay[budget:])
            free, far = (torch.as_tensor(x, device=weights.device) for x in (free, far))
            weights[b, h, free] = weights[b, h, far]
            weights[b, h, budget:] = 0
            moves.append((b, h, free, far))
    if case["bits"] == 16:
        rows = [x.double() for x in pages]
        for b, h, free, far in moves:
            for x in rows:
                x[table[b, free // page], h, free % page] = x[table[b, far // page], h, far % page]
        return {"lengths": None, "weights": weights, "positions": None, "key_pages": rows[0],
                "value_pages": rows[1]}
    rows = [torch.zeros(case["batch"], budget, kv, case["dim"], dtype=torch.float64,
                        device=weights.device) for _ in range(2)]
    for x, name in zip(rows, ("key", "value")):
        for b in range(case["batch"]):
            n = int(state["lengths"][b])
            if n < 0:
                continue
            held_rows = _rows(state, name, b, n)
            x[b, :min(n, budget)] = held_rows[:budget]
            for at, h, free, far in moves:
                if at == b:
                    x[b, free, h] = held_rows[far, h]
    return {"lengths": None, "weights": weights, "positions": None, "keys": rows[0],
            "values": rows[1]}
