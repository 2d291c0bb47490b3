"""Gathered attention weights and evictions of the paged cache against their definition in 64 bits."""

import math

import pytest
import torch

from exp3_amd import paged
import paged_reference as ref
import trees_reference as trees

pytestmark = pytest.mark.gpu

LAYOUTS = ((28, 4, 128), (16, 4, 256), (8, 8, 128), (20, 1, 128), (34, 2, 256))


# ------------------------------------------------------------------ weights

def _check_weights(s, scale, q=None, more=0, lse=None):
    cache, table, starts, counts = ref.on_gpu(s)
    queries = s.q.cuda() if q is None else q
    if lse is None:
        lse = paged.paged_attention(queries, cache, table, starts, scale, counts, return_lse=True)[1]
    reach = s.table.shape[1] * s.page
    kv = s.held[0].shape[1]
    gen = torch.Generator().manual_seed(1)
    before = torch.rand(s.batch, kv, reach + more, generator=gen) * 0.01
    weights = before.cuda()
    paged.accumulate_weights(weights, queries, lse, cache, table, starts, scale, counts)
    want, off = trees.gathered(s, lse.double().cpu(), scale)
    got = weights.double().cpu()
    assert torch.equal(got[..., reach:], before[..., reach:].double())
    total = want + before[..., :reach].double()
    wrong = (got[..., :reach] - total).abs() - off - 2.0 ** -24 * total
    assert wrong.max() <= 0, (wrong.max().item(), off.max().item())
    untouched = want == 0
    assert torch.equal(got[..., :reach][untouched], before[..., :reach][untouched].double())
    return weights, before


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("tokens", (1, 3, 9))
def test_weights_lengths(gpu, layout, tokens, bits):
    starts = (0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257, 300, -1)
    s = ref.make(61, len(starts), tokens, *layout, 16, 20, starts, bits=bits, sharp=2.0, spare=0)
    _check_weights(s, layout[2] ** -0.5, more=tokens % 2)


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("tokens,layout,starts", ((33, (28, 4, 128), (0, 200)), (64, (16, 4, 256), (5, 130)),
                                                  (150, (8, 2, 128), (0, 100)), (300, (4, 1, 128), (0, 20))))
def test_weights_of_many_tokens(gpu, tokens, layout, starts, bits):
    """Several chunks of columns; prompts from their first token on, which see each other in part."""
    s = ref.make(62, 2, tokens, *layout, 32, 11, starts, bits=bits, spare=0)
    _check_weights(s, 0.08)


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("tokens", (4, 90))
def test_weights_empty_rows(gpu, tokens, bits):
    """Free slots, padding, the table's end, pages outside the cache, starts next to 2^31."""
    s = ref.make(63, 9, tokens, 14, 2, 128, 16, 20, (-1, 100, 150, 318, 77, 50, 2**31 - 2, -9, 0),
                 counts=(tokens, 2, 0, tokens, tokens, tokens, tokens, tokens, -1), bits=bits)
    s.table[1, 3], s.table[4, :], s.table[5, 3] = -1, 2**31 - 1, s.pages
    _check_weights(s, 0.1)


def test_weights_long(gpu):
    s = ref.make(64, 2, 2, 4, 2, 128, 128, 100, (12700, 9000), sharp=3.0, spare=0)
    _check_weights(s, 0.09)


@pytest.mark.parametrize("scale", (-0.2, 0.0, 1.5))
def test_weights_scales(gpu, scale):
    _check_weights(ref.make(65, 2, 3, 8, 2, 128, 16, 8, (100, 3)), scale)


def test_weights_special_rows(gpu):
    """An LSE of -inf adds nothing, whatever the scores; NaN in a row that is no token, or behind the
    last key, neither; a NaN key gathers NaN, alone."""
    s = ref.make(66, 2, 4, 8, 2, 128, 16, 8, (60, 20), counts=(4, 2))
    lse = torch.full((2, 4, 8), 1.0)
    lse[0, 1], lse[1, 2:] = -math.inf, math.nan
    s.q[1, 2:] = math.nan
    for x in s.held:
        x[int(s.table[0, 4]), :, 0] = math.nan           # position 64, behind the last
    _check_weights(s, 0.1, lse=lse.cuda())
    s.held[0][int(s.table[0, 0]), 1, 5] = math.nan
    cache, table, starts, counts = ref.on_gpu(s)
    weights = torch.zeros(2, 2, 128, device="cuda")
    paged.accumulate_weights(weights, s.q.cuda(), lse.cuda(), cache, table, starts, 0.1, counts)
    nan = torch.isnan(weights).nonzero().tolist()
    assert nan == [[0, 1, 5]]


@pytest.mark.parametrize("tokens", (30, 160))
def test_weights_special_rows_of_many_tokens(gpu, tokens):
    """The same where the columns are many; a row of NaN whose LSE is -inf."""
    s = ref.make(68, 2, tokens, 8, 2, 128, 16, 50, (560, 20), counts=(tokens, tokens // 2))
    lse = torch.full((2, tokens, 8), 1.0)
    lse[0, 1], lse[0, 17, 3], lse[1, tokens // 2:] = -math.inf, -math.inf, math.nan
    s.q[0, 1] = s.q[1, tokens // 2:] = math.nan
    behind = 560 + tokens
    for x in s.held:
        x[int(s.table[0, behind // 16]), :, behind % 16:] = math.nan
    _check_weights(s, 0.1, lse=lse.cuda())
    s.held[0][int(s.table[0, 33]), 1, 5] = math.nan
    cache, table, starts, counts = ref.on_gpu(s)
    weights = torch.zeros(2, 2, 800, device="cuda")
    paged.accumulate_weights(weights, s.q.cuda(), lse.cuda(), cache, table, starts, 0.1, counts)
    assert torch.isnan(weights).nonzero().tolist() == [[0, 1, 533]]


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("tokens,layout", ((100, (16, 4, 256)), (140, (16, 4, 256)), (140, (28, 4, 128)),
                                           (70, (28, 4, 128)), (3, (16, 4, 256)), (2, (28, 4, 128))))
def test_weights_of_several_blocks(gpu, tokens, layout, bits):
    """Blocks of keys that one workgroup has and that workgroups share; ragged, with padding."""
    s = ref.make(69, 5, tokens, *layout, 64, 30, (1500, 511 - tokens, -1, 900, 0),
                 counts=(tokens, tokens, tokens, tokens - 1, tokens), bits=bits)
    first, before = _check_weights(s, 0.08, more=2)
    again, _ = _check_weights(s, 0.08, more=2)
    assert torch.equal(first, again)


def test_weights_strided_queries_and_sums(gpu):
    """Queries read in place; a row's weights sum to its number of query heads and tokens."""
    s = ref.make(67, 2, 5, 12, 2, 128, 16, 20, (300, 100))
    fused = torch.cat((s.q, s.k, s.v), 2).cuda()
    weights, before = _check_weights(s, 0.1, q=fused[:, :, :12])
    again, _ = _check_weights(s, 0.1)
    assert torch.equal(weights, again)
    grown = (weights.double().cpu() - before.double()).sum(-1)
    assert (grown - 5 * 6).abs().max() <= 1e-3


# ----------------------------------------------------------------- evictions

def _ledger(seed, s, slots, moved):
    """Weights with ties, zeros, infinities and NaN; positions of the first `moved` slots."""
    gen = torch.Generator().manual_seed(seed)
    kv = s.held[0].shape[1]
    weights = torch.randint(0, 40, (s.batch, kv, slots), generator=gen).float() * 0.25
    fine = torch.rand(s.batch, kv, slots, generator=gen)
    weights = torch.where(fine < 0.5, weights, torch.exp(5 * torch.randn(weights.shape, generator=gen)))
    weights[fine < 0.02] = math.nan
    weights[(fine > 0.02) & (fine < 0.04)] = -0.0
    weights[(fine > 0.04) & (fine < 0.05)] = math.inf
    weights[(fine > 0.05) & (fine < 0.06)] = -1.0
    positions = None
    if moved:
        positions = torch.full(weights.shape, -1, dtype=torch.int32)
        for b in range(s.batch):
            for h in range(kv):
                positions[b, h, :moved] = torch.randperm(2 * moved, generator=gen)[:moved]
    return weights, positions


def _check_evict(s, lengths, budget, recent=0, sinks=0, seen=None, moved=0, more=0, in_place=False):
    slots = s.table.shape[1] * s.page + more
    weights, positions = _ledger(7, s, slots, moved)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    seen = None if seen is None else torch.tensor(seen, dtype=torch.int32)
    want = trees.evict(s, lengths, weights, budget, positions, seen, recent, sinks)
    cache, table, _, _ = ref.on_gpu(s)
    w, p = weights.cuda(), None if positions is None else positions.cuda()
    out = None
    if in_place:
        out = (w, p if p is not None else torch.empty_like(w, dtype=torch.int32))
    got = paged.evict_tokens(cache, table, lengths.cuda(), w, budget, p,
                             None if seen is None else seen.cuda(), recent, sinks, out)
    assert torch.equal(got[0].cpu(), want[0])
    torch.testing.assert_close(got[1].cpu(), want[1], rtol=0, atol=0, equal_nan=True)
    assert torch.equal(got[2].cpu(), want[2])
    for x, y in zip(ref.contents(cache), want[3:]):
        assert torch.equal(x, y.double())
    if in_place:
        assert got[1].data_ptr() == w.data_ptr() and got[2].data_ptr() == out[1].data_ptr()
    else:
        torch.testing.assert_close(w.cpu(), weights, rtol=0, atol=0, equal_nan=True)
        assert p is None or torch.equal(p.cpu(), positions)


@pytest.mark.parametrize("in_place", (False, True))
@pytest.mark.parametrize("bits,dim,page", ((16, 128, 16), (4, 128, 32), (16, 256, 64), (4, 256, 16)))
@pytest.mark.parametrize("budget,recent,sinks", ((1, 0, 0), (1, 1, 0), (20, 5, 2), (64, 64, 0), (100, 0, 7),
                                                 (191, 20, 4)))
def test_evict(gpu, budget, recent, sinks, bits, dim, page, in_place):
    """Lengths around the budget, free slots, none; the first eviction and a later one."""
    lengths = (0, 1, -1, 20, 21, 63, 64, 65, 100, 101, 128, 190, 191, 192)
    s = ref.make(71, len(lengths), 1, 4, 2, dim, page, 192 // page, lengths, bits=bits)
    _check_evict(s, lengths, budget, recent, sinks, in_place=in_place, more=3)
    _check_evict(s, lengths, budget, recent, sinks, [max(n, 0) * 3 + 200 for n in lengths], moved=20,
                 in_place=in_place)


@pytest.mark.parametrize("keys,budget", ((1500, 700), (3000, 100), (5000, 4999), (2049, 1025),
                                         (4097, 2000), (32768, 9000), (33001, 20000), (50000, 300)))
def test_evict_long(gpu, keys, budget):
    """Rows of several digits' walks: ranks in LDS (up to 4096 and 32768 slots) and formed anew."""
    s = ref.make(72, 2, 1, 2, 1, 128, 64, -(-keys // 64), (0, 0))
    _check_evict(s, (keys, keys - 333), budget, budget // 10, 3)


@pytest.mark.parametrize("keys", (700, 9000, 40000))
@pytest.mark.parametrize("value", (0.0, 1.5, math.nan))
def test_evict_ties(gpu, keys, value):
    """All weights alike, or all but a few: the lowest slots stay."""
    s = ref.make(78, 1, 1, 1, 1, 128, 128, -(-keys // 128), (0,))
    cache, table, _, _ = ref.on_gpu(s)
    weights = torch.full((1, 1, s.table.shape[1] * 128), value, device="cuda")
    lengths = torch.tensor([keys], dtype=torch.int32, device="cuda")
    budget = keys // 2
    left, _, positions = paged.evict_tokens(cache, table, lengths, weights, budget, recent=10)
    want = list(range(budget - 10)) + list(range(keys - 10, keys))
    assert int(left[0]) == budget and positions[0, 0, :budget].tolist() == want
    weights[0, 0, keys - 100:keys - 50:2] = math.inf
    positions = paged.evict_tokens(cache, table, lengths, weights, budget)[2]
    assert positions[0, 0, :budget].tolist() == \
        list(range(budget - 25)) + list(range(keys - 100, keys - 50, 2))


def test_evict_left_alone(gpu):
    """Sequences with a token that has no place, longer than the table reaches, next to 2^31; a place
    that is missing behind the length does not count."""
    s = ref.make(73, 5, 1, 4, 2, 128, 16, 6, (0,) * 5)
    s.table[0, 2], s.table[1, 4], s.table[4, 0] = -1, s.pages, 2**31 - 1
    _check_evict(s, (50, 50, 97, 2**31 - 1, 50), 20, 4, 2, more=4)


def test_evict_budget_of_the_reach(gpu):
    s = ref.make(74, 2, 1, 4, 2, 128, 16, 4, (0, 0))
    _check_evict(s, (64, 30), 64, 4, 2)
    _check_evict(s, (64, 30), 2**31 - 1, 4, 2)


def test_evict_again_is_nothing(gpu):
    s = ref.make(75, 2, 1, 4, 2, 128, 16, 10, (0, 0))
    cache, table, _, _ = ref.on_gpu(s)
    weights, _ = _ledger(8, s, 160, 0)
    lengths = torch.tensor([160, 90], dtype=torch.int32, device="cuda")
    first = paged.evict_tokens(cache, table, lengths, weights.cuda(), 40, recent=8)
    pages = cache.key_pages.clone(), cache.value_pages.clone()
    second = paged.evict_tokens(cache, table, *first[:2], 40, first[2], lengths, recent=8)
    for x, y in zip(first, second):
        torch.testing.assert_close(x, y, rtol=0, atol=0, equal_nan=True)
    assert torch.equal(cache.key_pages, pages[0]) and torch.equal(cache.value_pages, pages[1])


# ------------------------------------------------------------------- together

@pytest.mark.parametrize("bits", (16, 4))
def test_decode_with_evictions(gpu, bits):
    """Steps of append, attention and weights with an eviction every few, against attention over the
    tokens that are kept, whose positions the ledger names."""
    heads, kv, dim, scale, budget = 8, 2, 128, 0.09, 24
    gen = torch.Generator().manual_seed(76)
    cache = paged.empty_pages(12, 16, kv, dim, "cuda", four_bit=bits == 4)
    for x in (cache.key_pages, cache.value_pages, cache.key_scales, cache.value_scales):
        if x is not None:
            x.zero_()
    table = torch.randperm(12, generator=gen)[:4].view(2, 2).int().cuda()
    rope = paged.rope_table(200, dim, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    text = torch.zeros(2, dtype=torch.int32, device="cuda")
    weights, positions = torch.zeros(2, kv, 32, device="cuda"), None
    tokens = []                                              # K and V as they were stored
    for step in range(60):
        q, k, v = (torch.randn(2, 1, n, dim, generator=gen).to(torch.bfloat16).cuda()
                   for n in (heads, kv, kv))
        turned, _ = paged.append_tokens(cache, table, lengths, k, v, q, rope, positions=text[:, None])
        stored = paged.gather_tokens(cache, table, lengths, 1)
        tokens.append([x[:, 0].double().cpu() for x in stored])
        out, lse = paged.paged_attention(turned, cache, table, lengths, scale, return_lse=True)
        n = int(lengths[0]) + 1
        for b in range(2):
            for h in range(heads):
                g = h // (heads // kv)
                at = [step + 1 - n + p for p in range(n)] if positions is None else \
                    [int(x) if x >= 0 else step + 1 - n + p
                     for p, x in enumerate(positions[b, g, :n].tolist())]
                keys = torch.stack([tokens[p][0][b, g] for p in at])
                values = torch.stack([tokens[p][1][b, g] for p in at])
                p = torch.softmax(keys @ turned[b, 0, h].double().cpu() * scale, 0)
                want = p @ values
                # the output's half step and, of |q| |k| below 2^9, 2^-13 of P |V|
                off = (out[b, 0, h].double().cpu() - want).abs() - 2.0 ** -8 * want.abs()
                assert off.max() <= 2.0 ** -13 * float((p @ values.abs()).max())
        paged.accumulate_weights(weights, turned, lse, cache, table, lengths, scale)
        lengths, text = lengths + 1, text + 1
        if n == 32:
            lengths, weights, positions = paged.evict_tokens(cache, table, lengths, weights, budget,
                                                             positions, text, recent=6, sinks=2)
            kept = positions[0, 0, :budget].tolist()
            assert set(range(2)) <= set(kept) and set(range(step - 5, step + 1)) <= set(kept)
            assert len(set(kept)) == budget
    assert positions is not None and int(lengths[0]) <= 32


def test_eviction_in_a_graph(gpu):
    """A captured step with weights and an eviction in place, replayed and compared with eager calls."""
    s = ref.make(77, 3, 2, 28, 4, 128, 16, 16, (100, 130, -1))
    cache, table, starts, _ = ref.on_gpu(s)
    weights = torch.rand(3, 4, 256, device="cuda")
    positions = torch.full((3, 4, 256), -1, dtype=torch.int32, device="cuda")
    q = s.q.cuda()

    def step(cache, starts, weights, positions):
        out, lse = paged.paged_attention(q, cache, table, starts, 0.1, return_lse=True)
        paged.accumulate_weights(weights, q, lse, cache, table, starts, 0.1)
        held = torch.where(starts < 0, -1, starts + 2).int()
        return (out, *paged.evict_tokens(cache, table, held, weights, 90, positions, None, 10, 2,
                                         (weights, positions)))

    step(cache, starts, weights, positions)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(cache, starts, weights, positions)
    for round in range(4):
        gen = torch.Generator().manual_seed(round)
        starts.copy_(torch.tensor([(100, 130, -1), (0, 254, 88), (89, 60, 200), (-1, 100, 100)][round]))
        pages = torch.randn(s.held[0].shape, generator=gen).to(torch.bfloat16)
        eager = paged.PagedCache(pages.cuda(), pages.cuda() + 1)
        cache.key_pages.copy_(eager.key_pages)
        cache.value_pages.copy_(eager.value_pages)
        weights.copy_(torch.rand(weights.shape, generator=gen))
        positions.fill_(-1)
        other = weights.clone(), positions.clone()
        torch.cuda.synchronize()
        graph.replay()
        want = step(eager, starts, *other)
        torch.cuda.synchronize()
        for x, y in zip(captured, want):
            assert torch.equal(x, y)
        assert torch.equal(cache.key_pages, eager.key_pages)
        assert torch.equal(cache.value_pages, eager.value_pages)
