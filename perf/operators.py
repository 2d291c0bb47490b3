"""Cases of the paged KV cache: appending tokens with the rotary embedding applied on the
way, reading tokens back, and attention of new tokens over the pages, with pages in
bfloat16 or in 4 bits.

A page holds ``page_size`` tokens of every KV head, ``[pages, Hkv, page_size, D]``; a
sequence's tokens are found through its row of the page table. 4-bit pages hold E2M1
values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two per byte with the even dim in the low
half, and one power-of-two scale (E8M0, bias 127) per token, head and 32 dims.

``run`` computes a case in plain torch operations, or, with ``own`` set, through
``exp3_amd.paged``.
"""

from __future__ import annotations

import math

import torch

own = False

GROUP = 32                      # dims per scale of a 4-bit page
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# (query heads, KV heads, head dim, rotated dims): Qwen2.5-7B, Llama-like 4:1, Qwen2.5-1.5B,
# no GQA, and the Qwen3.5 full-attention layers, which rotate a quarter of the dims
LAYOUTS = ((28, 4, 128, 128), (32, 8, 128, 128), (12, 2, 128, 128), (8, 8, 128, 128),
           (16, 4, 256, 64))


def _case(op, keys, layout=LAYOUTS[0], batch=1, tokens=1, bits=16, page=16, ragged=False, **more):
    """keys: those of the longest sequence, its new tokens among them; tokens: new ones per
    sequence. Ragged batches have shorter sequences and, from four sequences on, a free slot."""
    return dict(op=op, keys=keys, batch=batch, tokens=tokens, bits=bits, page=page, ragged=ragged,
                q_heads=layout[0], kv_heads=layout[1], dim=layout[2], rotary=layout[3], **more)


def listed():
    return [
        # one decode step of one chat: launches and latency
        _case("append", 1090, name="append_decode_1"),
        # one decode step of a full serving batch into 4-bit pages, read back as values
        _case("append", 8192, LAYOUTS[1], batch=64, bits=4, page=128, ragged=True,
              name="append_decode_b64_4bit"),
        # a whole 32K prompt; the prefill attention takes the rotated queries and keys
        _case("append", 32640, tokens=32640, page=128, name="append_prompt_32640"),
        # padded prompts behind cached prefixes, a quarter of 256 dims rotated, 4-bit pages
        _case("append", 6209, LAYOUTS[4], batch=4, tokens=2113, bits=4, page=64, ragged=True,
              name="append_prompts_b4_4bit"),
        # a cached prefix read back for a prefill that continues it
        _case("gather", 8191, tokens=8191, bits=4, page=16, name="gather_4bit_8191"),
        # four conversations of unlike lengths
        _case("gather", 12001, LAYOUTS[1], batch=4, tokens=12001, page=128, ragged=True,
              name="gather_b4_12001"),
        # attention of a decode step behind a short prompt
        _case("attention", 1090, name="attention_1090"),
        # a batch of long conversations of unlike lengths
        _case("attention", 16000, LAYOUTS[1], batch=8, page=128, ragged=True,
              name="attention_b8_16000"),
        # behind a 32K prompt in 4 bits
        _case("attention", 32641, bits=4, page=128, name="attention_4bit_32641"),
        # a full serving batch in 4 bits
        _case("attention", 8192, LAYOUTS[1], batch=64, bits=4, page=16, ragged=True,
              name="attention_4bit_b64_8192"),
        # four drafted tokens per sequence verified at once, head dim 256
        _case("attention", 12001, LAYOUTS[4], batch=4, tokens=4, bits=4, page=64, ragged=True,
              name="attention_4bit_d256_t4"),
        # the longest context
        _case("attention", 131072, bits=4, page=128, name="attention_4bit_131072"),
    ]


def _length(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(("append", "append", "gather", "attention", "attention", "attention"))
    layout = rng.choice(LAYOUTS)
    bits, page = rng.choice((16, 4)), rng.choice((16, 32, 64, 128))
    ragged = rng.random() < 0.5
    row = layout[1] * layout[2]                    # elements of one token's keys
    if op == "attention":
        batch = rng.choice((1, 1, 2, 3, 8, 24, 64))
        tokens = rng.choice((1, 1, 1, 2, 3, 5, 8))
        most = min(131072, (130_000_000 if bits == 16 else 400_000_000) // (row * batch))
        return _case(op, _length(rng, tokens, most), layout, batch, tokens, bits, page, ragged)
    if op == "append" and rng.random() < 0.4:      # decode steps
        batch, tokens = rng.choice((1, 2, 7, 33, 64)), rng.choice((1, 1, 2, 4))
        return _case(op, _length(rng, tokens, min(131072, 250_000_000 // (row * batch))), layout,
                     batch, tokens, bits, page, ragged)
    batch = rng.choice((1, 1, 2, 4))
    tokens = _length(rng, 2, 16_000_000 // (row * batch))
    if op == "gather":
        return _case(op, tokens, layout, batch, tokens, bits, page, ragged)
    return _case(op, tokens + rng.choice((0, 1, 100, 1000)), layout, batch, tokens, bits, page,
                 ragged)


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

def _rope_table(positions, rotary, device):
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * \
        1.0e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary)
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device).manual_seed(seed)
    batch, tokens, page = case["batch"], case["tokens"], case["page"]
    heads, kv, dim = case["q_heads"], case["kv_heads"], case["dim"]
    held, new = _plan(case)
    width = -(-case["keys"] // page)
    pages = batch * width + 3

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    # page ids as a server's free list leaves them: in no order
    table = torch.randperm(pages, generator=gen, device=device)[:batch * width]
    state = dict(case=case, scale=dim ** -0.5,
                 table=table.view(batch, width).to(torch.int32),
                 starts=torch.tensor(held, dtype=torch.int32, device=device),
                 new=torch.tensor([b * tokens + t for b in range(batch) for t in range(new[b])],
                                  device=device),
                 counts=torch.tensor(new, dtype=torch.int32, device=device)
                 if case["ragged"] else None)
    # keys with channels of unlike size, as projections with biases leave them
    gain = torch.exp(0.5 * normal(kv, 1, dim))
    for name, size in (("key", gain), ("value", 1.0)):
        held_pages, scales = [], []
        for part in torch.arange(pages, device=device).split(max(1, (1 << 27) // (kv * page * dim))):
            x = (normal(part.numel(), kv, page, dim) * size).to(torch.bfloat16)
            if case["op"] == "append":
                x.zero_()
            if case["bits"] == 4:
                x, scale = _to_4bit(x.float())
                scales.append(scale)
            held_pages.append(x)
        state[name + "_pages"] = torch.cat(held_pages)
        state[name + "_scales"] = torch.cat(scales) if scales else None
    if case["op"] == "append":
        # one projection's output: queries, keys and values side by side
        fused = normal(batch, tokens, heads + 2 * kv, dim)
        fused[:, :, heads:heads + kv] *= gain[:, 0]
        q, k, v = fused.to(torch.bfloat16).split((heads, kv, kv), 2)
        state |= dict(q=q, k=k, v=v, rope=_rope_table(width * page, case["rotary"], device),
                      keys=tokens > 8 and case["bits"] == 16)
    elif case["op"] == "attention":
        sharp = torch.linspace(0.3, 2.0, heads, device=device)[:, None]
        state["q"] = (normal(batch, tokens, heads, dim) * sharp).to(torch.bfloat16)
    return state


# -------------------------------------------------------------- plain forms

def _to_4bit(x):
    """[..., D] -> packed E2M1 values [..., D / 2] and E8M0 scales [..., D / 32]. The scale is
    that at which the largest value of its 32 lies in [3.5, 7) (it is clipped to 6 above
    that, at most one step of the grid); values round to nearest, ties to the even code. A
    value that is not finite makes its 32 NaN (scale 255)."""
    x = x.unflatten(-1, (-1, GROUP))
    top = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(top)
    scale = (exponent + (mantissa >= 0.875) + 124).clamp(2, 252)
    scale = torch.where(top == 0, 2, torch.where(torch.isfinite(top), scale, 255))
    y = torch.ldexp(x.abs(), (127 - scale).clamp(min=-125)[..., None])
    code = torch.zeros_like(y, dtype=torch.uint8)
    for border, up in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)):
        code += (y >= border) if up else (y > border)
    code |= (x < 0).to(torch.uint8) << 3
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] | code[..., 1] << 4, scale.to(torch.uint8)


def _from_4bit(packed, scale):
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    value = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=packed.device)[code.long()]
    size = torch.ldexp(torch.ones((), device=packed.device), scale.int() - 127)
    size = torch.where(scale == 255, math.nan, size)
    return (value.unflatten(-1, (-1, GROUP)) * size[..., None]).flatten(-2)


def _places(state):
    """[B, T] positions of the new tokens, whether each is a token, its page and its slot."""
    case, starts, table = state["case"], state["starts"].long(), state["table"]
    step = torch.arange(case["tokens"], device=starts.device)
    count = case["tokens"] if state["counts"] is None else state["counts"].long()[:, None]
    where = starts[:, None] + step
    live = (starts[:, None] >= 0) & (step < count) & (where < table.shape[1] * case["page"])
    where = torch.where(live, where, 0)
    return where, live, table.long().gather(1, where // case["page"]), where % case["page"]


def _rotated(x, cos, sin):
    """[B, T, H, D] with the first 2 x cos.shape[-1] dims rotated, halves paired."""
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)


def _plain_append(state):
    four = state["case"]["bits"] == 4
    where, live, page, slot = _places(state)
    page, slot = page.flatten()[state["new"]], slot.flatten()[state["new"]]
    cos, sin = (t[where][:, :, None] for t in state["rope"])
    empty = ~live[..., None, None]
    q = _rotated(state["q"].float(), cos, sin).masked_fill(empty, 0).to(torch.bfloat16)
    if four:     # values next to a border of the 4-bit grid: 64 bits
        k = _rotated(state["k"].double(), cos.double(), sin.double())
    else:
        k = _rotated(state["k"].float(), cos, sin).to(torch.bfloat16)
    for name, x in (("key", k), ("value", state["v"].double() if four else state["v"])):
        if four:
            x, scale = _to_4bit(x)
            state[name + "_scales"][page, :, slot] = scale.flatten(0, 1)[state["new"]]
        state[name + "_pages"][page, :, slot] = x.flatten(0, 1)[state["new"]]
    if four:
        return {"q": q, **_plain_gather(state)}
    rows = {"keys": k.masked_fill(empty, 0)} if state["keys"] else {}
    return {"q": q, "key_pages": state["key_pages"], "value_pages": state["value_pages"], **rows}


def _plain_gather(state):
    _, live, page, slot = _places(state)
    out = {}
    for name in ("key", "value"):
        x = state[name + "_pages"][page, :, slot]
        if state["case"]["bits"] == 4:
            x = _from_4bit(x, state[name + "_scales"][page, :, slot]).to(torch.bfloat16)
        out[name + "s"] = x.masked_fill(~live[..., None, None], 0)
    return out


def _plain_attention(state):
    case, q = state["case"], state["q"]
    batch, tokens, heads, dim = q.shape
    kv = case["kv_heads"]
    where, live, _, _ = _places(state)
    k, v = (state[name + "_pages"][state["table"].long()] for name in ("key", "value"))
    if case["bits"] == 4:
        k, v = (_from_4bit(x, state[name + "_scales"][state["table"].long()])
                for x, name in ((k, "key"), (v, "value")))
    k, v = (x.transpose(1, 2).reshape(batch, kv, -1, dim).float() for x in (k, v))
    rows = q.float().view(batch, tokens, kv, heads // kv, dim).permute(0, 2, 1, 3, 4)
    logits = (rows.reshape(batch, kv, -1, dim) @ k.transpose(2, 3) * state["scale"])
    logits = logits.view(batch, kv, tokens, heads // kv, -1)
    seen = live[..., None] & (torch.arange(k.shape[2], device=q.device) <= where[..., None])
    logits = logits.masked_fill(~seen[:, None, :, None], -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(torch.isinf(top), 0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1, total)
    out = (p.view(batch, kv, -1, k.shape[2]) @ v).view(batch, kv, tokens, heads // kv, dim)
    lse = (total.log() + top)[..., 0]
    return {"out": out.permute(0, 2, 1, 3, 4).reshape(q.shape).to(torch.bfloat16),
            "lse": lse.permute(0, 2, 1, 3).reshape(batch, tokens, heads)}


# ---------------------------------------------------------------------- run

def _own(state):
    from exp3_amd import paged

    case = state["case"]
    cache = paged.PagedCache(state["key_pages"], state["value_pages"], state["key_scales"],
                             state["value_scales"])
    place = (cache, state["table"], state["starts"])
    if case["op"] == "attention":
        out, lse = paged.paged_attention(state["q"], *place, state["scale"], state["counts"],
                                         return_lse=True)
        return {"out": out, "lse": lse}
    out = {}
    if case["op"] == "append":
        q, k = paged.append_tokens(*place, state["k"], state["v"], state["q"], state["rope"],
                                   state["counts"], return_keys=state["keys"])
        if case["bits"] == 16:
            rows = {"keys": k} if state["keys"] else {}
            return {"q": q, "key_pages": cache.key_pages, "value_pages": cache.value_pages, **rows}
        out["q"] = q
    out["keys"], out["values"] = paged.gather_tokens(*place, case["tokens"], state["counts"])
    return out


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "gather": _plain_gather,
            "attention": _plain_attention}[state["case"]["op"]](state)


# --------------------------------------------------------------------- work

def work(case):
    held, new = _plan(case)
    heads, kv, dim = case["q_heads"], case["kv_heads"], case["dim"]
    row = dim * 2 if case["bits"] == 16 else dim // 2 + dim // GROUP
    wide = case["batch"] * case["tokens"] * dim * 2       # bf16 rows of one head, padding too
    count = sum(new)
    if case["op"] == "append":
        size = 2 * heads * dim * count + 4 * kv * dim * count + heads * wide + 2 * kv * row * count
        size += 4 * case["rotary"] * count
        if case["bits"] == 4:
            size += 2 * kv * wide
        elif case["tokens"] > 8:
            size += kv * wide
        return {"bytes": size, "flops": 3 * case["rotary"] * (heads + kv) * count}
    if case["op"] == "gather":
        return {"bytes": 2 * kv * (row * count + wide), "flops": 0}
    keys = sum(h + n for h, n in zip(held, new) if h >= 0)
    pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new) if h >= 0)
    return {"bytes": 2 * kv * row * keys + 2 * heads * wide + 4 * heads * wide // (2 * dim),
            "flops": 4 * heads * dim * pairs}


# -------------------------------------------------------------------- exact

def _grid(x):
    """The 4-bit pages' value of every element of [..., 32] groups, from the nearest grid point."""
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    top = x.abs().max(-1, keepdim=True).values
    step = torch.full_like(top, 2.0 ** -125)
    fits = top > 0
    step[fits] = 2.0 ** torch.floor(torch.log2(top[fits] / 7.0) + 1)
    # log2 is not exact: put the largest value into [3.5, 7) steps
    step = torch.where(top >= 7 * step, 2 * step, step)
    step = torch.where((top < 3.5 * step) & (top > 0), step / 2, step)
    step = step.clamp(2.0 ** -125, 2.0 ** 125)
    off = (x.abs() / step)[..., None] - grid
    near = off.abs().min(-1, keepdim=True).values
    hit = off.abs() == near                                  # two at a tie: the even code
    even = torch.tensor([1, 0] * 4, dtype=torch.float64, device=x.device)
    code = (hit * (1 + even)).argmax(-1)
    return torch.copysign(grid[code] * step, x)


def _turn(x, cos, sin):
    """The rotation as a product of complex numbers."""
    half = cos.shape[-1]
    z = torch.complex(x[..., :half], x[..., half:2 * half]) * torch.complex(cos, sin)[:, None]
    return torch.cat((z.real, z.imag, x[..., 2 * half:]), -1)


def _value_rows(state, name, b, first, last):
    """[last - first, Hkv, D] in float64 of sequence b's tokens."""
    page = state["case"]["page"]
    at = torch.arange(first, last, device=state["table"].device)
    ids = state["table"][b].long()[torch.div(at, page, rounding_mode="floor")]
    rows = state[name + "_pages"][ids, :, at % page]
    if state["case"]["bits"] == 16:
        return rows.double()
    values = torch.tensor([(-1.0) ** (c >> 3) * E2M1[c & 7] for c in range(16)],
                          dtype=torch.float64, device=rows.device)
    pairs = torch.stack((values[(rows % 16).long()], values[(rows // 16).long()]), -1)
    exponent = state[name + "_scales"][ids, :, at % page].double() - 127
    return pairs.reshape(*rows.shape[:2], -1, GROUP).mul(2.0 ** exponent[..., None]).flatten(2)


def exact(case, seed):
    state = prepare(case, seed)
    held, new = _plan(case)
    batch, tokens, kv, dim = case["batch"], case["tokens"], case["kv_heads"], case["dim"]
    wide = dict(dtype=torch.float64, device=state["table"].device)
    if case["op"] == "attention":
        heads = case["q_heads"]
        out = torch.zeros(batch, tokens, heads, dim, **wide)
        lse = torch.full((batch, tokens, heads), -math.inf, **wide)
        for b in range(batch):
            if held[b] < 0:
                continue
            k = _value_rows(state, "key", b, 0, held[b] + new[b]).repeat_interleave(heads // kv, 1)
            v = _value_rows(state, "value", b, 0, held[b] + new[b]).repeat_interleave(heads // kv, 1)
            for t in range(new[b]):
                n = held[b] + t + 1
                logits = (k[:n] * state["q"][b, t].double()).sum(-1) * state["scale"]
                lse[b, t] = torch.logsumexp(logits, 0)
                out[b, t] = (torch.softmax(logits, 0)[..., None] * v[:n]).sum(0)
        return {"out": out, "lse": lse}
    rows = [torch.zeros(batch, tokens, kv, dim, **wide) for _ in range(2)]
    if case["op"] == "gather":
        for b in range(batch):
            for x, name in zip(rows, ("key", "value")):
                x[b, :new[b]] = _value_rows(state, name, b, held[b], held[b] + new[b])
        return {"keys": rows[0], "values": rows[1]}
    q = torch.zeros(batch, tokens, case["q_heads"], dim, **wide)
    cache = [state[name + "_pages"].double() for name in ("key", "value")] \
        if case["bits"] == 16 else []
    for b in range(batch):
        n, at = new[b], torch.arange(held[b], held[b] + new[b], device=q.device)
        cos, sin = (t[at].double() for t in state["rope"])
        q[b, :n] = _turn(state["q"][b, :n].double(), cos, sin)
        rows[0][b, :n] = _turn(state["k"][b, :n].double(), cos, sin)
        rows[1][b, :n] = state["v"][b, :n].double()
        for x, kept in zip(rows, cache):
            kept[state["table"][b].long()[at // case["page"]], :, at % case["page"]] = x[b, :n]
    if case["bits"] == 4:
        keys, values = (_grid(x.unflatten(-1, (-1, GROUP))).flatten(-2) for x in rows)
        return {"q": q, "keys": keys, "values": values}
    more = {"keys": rows[0]} if state["keys"] else {}
    return {"q": q, "key_pages": cache[0], "value_pages": cache[1], **more}
