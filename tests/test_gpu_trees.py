"""Drafted trees on the paged cache against their definition in 64 bits: the plan, attention of a
tree, appending at positions that are not places, acceptance and the moves of an accepted path."""

import pytest
import torch

from exp3_amd import paged
import paged_reference as ref
import trees_reference as trees

pytestmark = pytest.mark.gpu

LAYOUTS = ((28, 4, 128), (16, 4, 256), (8, 8, 128), (20, 1, 128), (34, 2, 256))


# --------------------------------------------------------------------- plan

@pytest.mark.parametrize("tokens", (1, 2, 3, 16, 63, 64, 65, 130, 256))
def test_draft_tree(gpu, tokens):
    parents = trees.random_parents(tokens, 5, tokens)
    parents[3] = torch.arange(tokens) - 1                          # a chain
    parents[4] = -1                                                # roots alone
    if tokens > 2:                                                 # no parents: behind a node, itself
        parents[4, 1], parents[4, 2] = 2, 2**31 - 1
        parents[2, 2] = -2**31
    seen, depth = trees.lineage(parents)
    depths, masks = paged.draft_tree(parents.cuda())
    assert torch.equal(depths.cpu(), depth) and torch.equal(masks.cpu(), trees.words(seen))


# ---------------------------------------------------------------- attention

def _check(s, seen, scale, max_keys=None, q=None):
    cache, table, starts, counts = ref.on_gpu(s)
    out, lse = paged.tree_attention(s.q.cuda() if q is None else q, cache, table, starts,
                                    trees.words(seen).cuda(), scale, counts, max_keys, return_lse=True)
    want, want_lse, out_off, lse_off = trees.tree_attention(s, seen, scale)
    out, lse = out.double().cpu(), lse.double().cpu()
    empty = torch.isinf(want_lse)
    assert (out[empty] == 0).all() and torch.equal(lse[empty], want_lse[empty])
    assert torch.isfinite(out).all()
    off = (out - want).abs() - 2.0 ** -8 * want.abs() - out_off
    assert off.max() <= 0, (off.max().item(), out_off.max().item())
    off = (lse - want_lse).abs()[~empty] - lse_off[~empty]
    assert off.numel() == 0 or off.max() <= 0, off.max().item()
    return out, lse


def _tree(seed, batch, tokens):
    return trees.lineage(trees.random_parents(seed, batch, tokens))[0]


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("tokens", (1, 2, 9, 23))
def test_tree_lengths(gpu, layout, tokens, bits):
    """One batch with prefixes of all sorts, none among them, and a free slot."""
    starts = (0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 255, 257, 511, 700, -1)
    s = ref.make(31, len(starts), tokens, *layout, 16, 48, starts, bits=bits, sharp=2.0, spare=0)
    _check(s, _tree(31, len(starts), tokens), layout[2] ** -0.5)


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("page", (32, 128, 1024))
def test_tree_pages(gpu, page, bits):
    s = ref.make(32, 3, 17, 28, 4, 128, page, -(-1500 // page), (1483, 77, 1023), bits=bits)
    seen = _tree(32, 3, 17)
    _check(s, seen, 0.1)
    _check(s, seen, 0.1, max_keys=1500)
    _check(s, seen, 0.1, max_keys=1)              # a wrong bound costs time, not results


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("batch,layout,keys,tokens", ((1, (4, 2, 128), 40001, 3),
                                                      (1, (2, 1, 256), 20003, 33),
                                                      (40, (8, 8, 128), 900, 5),
                                                      (3, (28, 4, 128), 6000, 20),
                                                      (2, (24, 3, 256), 3000, 19)))
def test_tree_long_and_wide(gpu, batch, layout, keys, tokens, bits):
    starts = tuple(max(0, keys - tokens - 41 * b) for b in range(batch))
    s = ref.make(33, batch, tokens, *layout, 64, -(-keys // 64), starts, bits=bits, sharp=4.0, spare=0)
    _check(s, _tree(33, batch, tokens), layout[2] ** -0.5)


@pytest.mark.parametrize("tokens,layout", ((64, (28, 4, 128)), (65, (16, 4, 256)), (130, (8, 8, 128)),
                                           (256, (6, 2, 128)), (200, (7, 1, 128))))
@pytest.mark.parametrize("bits", (16, 4))
def test_tree_many_tokens(gpu, tokens, layout, bits):
    """Several column tiles and words of a mask; trees behind nothing and behind a prefix that ends
    inside a unit."""
    s = ref.make(34, 3, tokens, *layout, 32, 20, (0, 33, 640 - tokens), bits=bits)
    _check(s, _tree(34, 3, tokens), 0.09)


@pytest.mark.parametrize("bits", (16, 4))
def test_tree_empty_rows(gpu, bits):
    """Free slots, padding, positions past the table, pages outside the cache (one in the middle,
    all of a sequence), starts next to 2^31."""
    s = ref.make(35, 9, 12, 14, 2, 128, 16, 20, (-1, 100, 250, 314, 77, 50, 2**31 - 2, -9, 0),
                 counts=(12, 7, 0, 12, 12, 12, 12, 12, -1), bits=bits)
    s.table[1, 3], s.table[4, :], s.table[5, 3] = -1, 2**31 - 1, s.pages
    _check(s, _tree(35, 9, 12), 0.1)


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("tokens", (40, 70))
def test_tree_any_masks(gpu, tokens, bits):
    """Random masks: nodes that do not see themselves, see later ones, or see nothing at all (a
    sequence without a prefix); bits of nodes that are not live count nothing."""
    gen = torch.Generator().manual_seed(36)
    seen = torch.rand(4, tokens, tokens, generator=gen) > 0.6
    seen[0, 3] = seen[0, 37] = False
    seen[1, 5] = False
    seen[2, :, :33] = False
    s = ref.make(36, 4, tokens, 12, 2, 128, 16, 20, (0, 21, 64, 0),
                 counts=(tokens, tokens, tokens - 1, 33), bits=bits)
    _, lse = _check(s, seen, 0.1)
    assert torch.isinf(lse[0, 3]).all() and torch.isfinite(lse[1, 5]).all()


@pytest.mark.parametrize("scale", (-0.2, 0.0, 3.0))
def test_tree_scales(gpu, scale):
    s = ref.make(37, 2, 7, 8, 2, 128, 16, 8, (100, 3))
    _check(s, _tree(37, 2, 7), scale)


def test_tree_strided_queries(gpu):
    s = ref.make(38, 2, 6, 6, 2, 128, 16, 8, (100, 3))
    seen = _tree(38, 2, 6)
    want, _ = _check(s, seen, 0.1)
    fused = torch.cat((s.q, s.k, s.v), 2).cuda()
    assert torch.equal(_check(s, seen, 0.1, q=fused[:, :, :6])[0], want)
    odd = torch.zeros(2, 6, 6, 129, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(s.q)
    assert torch.equal(_check(s, seen, 0.1, q=odd)[0], want)
    assert torch.equal(_check(s, seen, 0.1, q=torch._neg_view(-s.q.cuda()))[0], want)


@pytest.mark.parametrize("tokens", (8, 40))
@pytest.mark.parametrize("bits", (16, 4))
def test_tree_values_that_are_not_finite(gpu, bits, tokens):
    """NaN and infinities in places that nothing sees, or that some nodes do not see, do not reach
    those that do not; infinite values reach the others as they are."""
    s = ref.make(39, 2, tokens, 28, 4, 128, 16, 20, (150, 0), bits=bits, spare=0)
    seen = torch.eye(tokens, dtype=torch.bool)[None].repeat(2, 1, 1)      # no node sees another
    seen[:, 5] |= seen[:, 3]
    clean, _ = _check(s, seen, 0.1)
    cache, table, starts, _ = ref.on_gpu(s)
    position = 150 + 3
    page, slot = int(s.table[0, position // 16]), position % 16
    past = [(int(s.table[0, p // 16]), p % 16) for p in range(150 + tokens, 320)]
    if bits == 16:
        cache.value_pages[page, :, slot, 0] = float("inf")
        cache.value_pages[page, :, slot, 1] = float("nan")
        for a, b in past:
            cache.value_pages[a, :, b] = float("nan")
            cache.key_pages[a, :, b] = float("nan")
    else:
        cache.value_scales[page, :, slot] = 255
        for a, b in past:
            cache.value_scales[a, :, b] = 255
            cache.key_scales[a, :, b] = 255
    got = paged.tree_attention(s.q.cuda(), cache, table, starts, trees.words(seen).cuda(), 0.1)
    got = got.double().cpu()
    touched = torch.zeros(2, tokens, dtype=torch.bool)
    touched[0, 3] = touched[0, 5] = True
    off = (got[~touched] - clean[~touched]).abs()
    assert off.max() <= 2.0 ** -7 * clean.abs().max()
    if bits == 16:
        assert torch.isinf(got[0, [3, 5], :, 0]).all() and torch.isnan(got[0, [3, 5], :, 1]).all()
        assert torch.isfinite(got[0, [3, 5], :, 2:]).all()
    else:
        assert torch.isnan(got[0, [3, 5]]).all()


def test_tree_keys_that_are_not_finite(gpu):
    """A NaN key makes the rows that see it NaN, also where it is all that a part of the work sees;
    a key of -inf score counts nothing."""
    s = ref.make(40, 1, 4, 4, 2, 128, 16, 300, (4700,), spare=0)
    seen = torch.eye(4, dtype=torch.bool)[None]
    cache, table, starts, _ = ref.on_gpu(s)
    page = int(s.table[0, 4702 // 16])
    cache.key_pages[page, :, 4702 % 16] = float("nan")
    out, lse = paged.tree_attention(s.q.cuda(), cache, table, starts, trees.words(seen).cuda(), 0.1,
                                    return_lse=True)
    assert torch.isnan(out[0, 2]).all() and torch.isnan(lse[0, 2]).all()
    assert torch.isfinite(out[0, [0, 1, 3]]).all() and torch.isfinite(lse[0, [0, 1, 3]]).all()
    s = ref.make(41, 1, 2, 4, 2, 128, 16, 4, (0,), spare=0)
    s.q = s.q.abs() + 1
    s.held[0][int(s.table[0, 0]), :, 1] = -float("inf")
    cache, table, starts, _ = ref.on_gpu(s)
    both = torch.tensor([[[1], [2]]]).cuda()
    out, lse = paged.tree_attention(s.q.cuda(), cache, table, starts, both, 0.1, return_lse=True)
    assert torch.isfinite(out[0, 0]).all() and (out[0, 1] == 0).all() and torch.isinf(lse[0, 1]).all()


def test_chain_is_paged_attention(gpu):
    """A tree without branches sees what paged_attention does: two roundings of one value."""
    s = ref.make(42, 3, 6, 28, 4, 128, 64, 40, (2000, 77, 0), bits=4)
    cache, table, starts, _ = ref.on_gpu(s)
    chain = (torch.arange(6) - 1).int().repeat(3, 1).cuda()
    got, lse = paged.tree_attention(s.q.cuda(), cache, table, starts, paged.draft_tree(chain)[1], 0.1,
                                    return_lse=True)
    want, want_lse = paged.paged_attention(s.q.cuda(), cache, table, starts, 0.1, return_lse=True)
    # both are within half a step and 2^-14 of the largest value (4 bits: 6 x 2) of the exact one
    assert ((got - want).abs().double() <= 2.0 ** -7 * want.abs().double() + 2.0 ** -9).all()
    assert (lse - want_lse).abs().max() <= 2.0 ** -18 * (1 + want_lse.abs().max())


# ------------------------------------------------------- append at positions

@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("dim,rotary", ((128, 128), (128, 48), (256, 64)))
def test_append_at_positions(gpu, dim, rotary, interleaved, bits):
    """Rotated by the given positions, stored in the places; the table of angles is the text's."""
    s = ref.make(43, 3, 7, 6, 2, dim, 16, 4, (0, 30, 57), bits=bits)
    gen = torch.Generator().manual_seed(43)
    at = torch.randint(0, 5000, (3, 7), generator=gen).int()
    rope = paged.rope_table(5000, rotary)
    cache, table, starts, _ = ref.on_gpu(s)
    q, k = paged.append_tokens(cache, table, starts, s.k.cuda(), s.v.cuda(), s.q.cuda(),
                               tuple(x.cuda() for x in rope), interleaved=interleaved,
                               return_keys=True, positions=at.cuda())
    cos, sin = (x[at.long()][:, :, None].double() for x in rope)
    for got, x in ((q, s.q), (k, s.k)):
        want = ref.rotated(x.double(), cos, sin, interleaved)
        off = (got.double().cpu() - want).abs() - 2.0 ** -8 * want.abs()
        off[2] = 0          # its last token's place is past the table
        assert off.max() <= 2.0 ** -22 * 8
    turned = ref.rotated(s.k.double(), cos, sin, interleaved)
    key, value = ref.contents(cache)
    for b in range(3):
        for i in range(7):
            p = ref.live_position(s, b, i)
            if p is None:
                assert (q[b, i] == 0).all()
                continue
            page, slot = ref.place(s, b, p)
            assert torch.equal(value[page, :, slot], ref.four_bit(s.v[b, i]) if bits == 4
                               else s.v[b, i].double())
            if bits == 4:
                assert torch.equal(key[page, :, slot], ref.four_bit(turned[b, i]))
            else:
                assert torch.equal(key[page, :, slot], k[b, i].double().cpu())
    same = ref.on_gpu(s)[0]
    places = (s.starts[:, None] + torch.arange(7)).int().cuda()
    paged.append_tokens(same, table, starts, s.k.cuda(), s.v.cuda(), None,
                        tuple(x.cuda() for x in rope), interleaved=interleaved, positions=places)
    want = ref.on_gpu(s)[0]
    paged.append_tokens(want, table, starts, s.k.cuda(), s.v.cuda(), None,
                        tuple(x.cuda() for x in rope), interleaved=interleaved)
    assert torch.equal(same.key_pages, want.key_pages)


@pytest.mark.parametrize("bits", (16, 4))
def test_append_at_positions_past_the_angles(gpu, bits):
    s = ref.make(44, 1, 4, 4, 2, 128, 16, 2, (3,), bits=bits)
    rope = tuple(x.cuda() for x in paged.rope_table(10, 64))
    cache, table, starts, _ = ref.on_gpu(s)
    at = torch.tensor([[9, 10, -1, 2**31 - 1]], dtype=torch.int32, device="cuda")
    q, k = paged.append_tokens(cache, table, starts, s.k.cuda(), s.v.cuda(), s.q.cuda(), rope,
                               return_keys=True, positions=at)
    assert torch.isfinite(q[0, 0]).all()
    assert torch.isnan(q[0, 1:, :, :64]).all() and torch.isfinite(q[0, 1:, :, 64:]).all()
    key, value = ref.contents(cache)
    page = int(s.table[0, 0])
    assert torch.isnan(key[page, :, 4:7, :64]).all() and torch.isfinite(key[page, :, 3]).all()
    assert torch.isfinite(key[page, :, 4:7, 64:]).all() and torch.isfinite(value).all()


# --------------------------------------------------------------- acceptance

def _layers(s, count, seed):
    """Caches of several layers over one page table, and their contents on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    caches, held = [], []
    for _ in range(count):
        if s.bits == 4:
            raw = [torch.randint(0, 256, x.shape, generator=gen, dtype=torch.uint8)
                   for x in (*s.raw, *s.scales)]
            raw[2:] = [x % 100 + 80 for x in raw[2:]]
            caches.append(paged.PagedCache(*(x.cuda() for x in raw)))
        else:
            raw = [torch.randn(x.shape, generator=gen).to(torch.bfloat16) for x in s.held]
            caches.append(paged.PagedCache(*(x.cuda() for x in raw)))
        held.append(raw)
    return caches, held


def _same(caches, held):
    for cache, want in zip(caches, held):
        got = [x for x in (cache.key_pages, cache.value_pages, cache.key_scales, cache.value_scales)
               if x is not None]
        for x, y in zip(got, want):
            assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("bits,dim", ((16, 128), (4, 128), (16, 256), (4, 256)))
@pytest.mark.parametrize("tokens,layers", ((1, 1), (5, 3), (33, 35), (64, 2), (100, 1), (256, 1)))
def test_accept_drafts(gpu, tokens, layers, bits, dim):
    """Trees of every depth, free slots, padding, the table's end, pages outside the cache."""
    starts = (0, 13, -1, 40, 320 - tokens // 2 - 1, 31, 2**31 - 2)
    counts = (tokens, tokens, tokens, max(tokens - 2, 0), tokens, 0, tokens)
    s = ref.make(45, 7, tokens, 4, 2, dim, 16, 20, starts, counts, bits=bits)
    s.table[3, 3] = -1
    parents = trees.random_parents(45 + tokens, 7, tokens)
    parents[1] = torch.arange(tokens) - 1                          # a chain, all of it accepted
    gen = torch.Generator().manual_seed(46)
    drafts = torch.randint(0, 2, (7, tokens), generator=gen) + 2**40 * torch.randint(
        0, 2, (7, tokens), generator=gen)
    targets = torch.randint(0, 2, (7, tokens), generator=gen) + 2**40 * torch.randint(
        0, 2, (7, tokens), generator=gen)
    targets[1, :-1] = drafts[1, 1:]
    caches, held = _layers(s, layers, 47)
    _, table, starts, counts = ref.on_gpu(s)
    accepted, path, following = paged.accept_drafts(caches if layers > 1 else caches[0], table, starts,
                                                    parents.cuda(), drafts.cuda(), targets.cuda(), counts)
    longest = 0
    for b in range(7):
        live = trees.live_tokens(s, b)
        want = trees.accept(parents[b], drafts[b], targets[b], live)
        longest = max(longest, len(want))
        assert int(accepted[b]) == len(want)
        assert path[b].tolist() == want + [-1] * (tokens - len(want))
        assert int(following[b]) == (int(targets[b, want[-1]]) if want else -1)
        for raw in held:
            trees.move(s, raw, b, [(int(s.starts[b]) + j, int(s.starts[b]) + i)
                                   for j, i in enumerate(want)])
    assert longest == tokens
    _same(caches, held)


@pytest.mark.parametrize("bits", (16, 4))
def test_keep_path(gpu, bits):
    """Given paths: skipping nodes, from the first one on or not, ended by -1, by an index that does
    not ascend, or by one that is not live; the next row's source may be the last row's target."""
    paths = torch.full((7, 70), -1, dtype=torch.int32)
    paths[0, :4] = torch.tensor([0, 2, 5, 69])
    paths[1, :70] = torch.arange(70)
    paths[2, :5] = torch.tensor([1, 2, 3, 4, 4])
    paths[3, :3] = torch.tensor([3, 2, 9])
    paths[4, :4] = torch.tensor([0, 7, 30, 31])                    # 30 live tokens
    paths[5, :66] = torch.arange(4, 70)
    s = ref.make(48, 7, 70, 4, 2, 128, 32, 8, (5, 0, 31, 64, 7, 100, -1),
                 (70, 70, 70, 70, 30, 70, 70), bits=bits)
    caches, held = _layers(s, 2, 49)
    _, table, starts, counts = ref.on_gpu(s)
    assert paged.keep_path(caches, table, starts, paths.cuda(), counts) is None
    for b, want in enumerate(([0, 2, 5, 69], range(70), [1, 2, 3, 4], [3], [0, 7], range(4, 70), [])):
        for raw in held:
            trees.move(s, raw, b, [(int(s.starts[b]) + j, int(s.starts[b]) + i)
                                   for j, i in enumerate(want)])
    _same(caches, held)


# ------------------------------------------------------------------- streams

def test_tree_step_in_a_graph(gpu):
    """A captured step of two trees, replayed with other lengths, drafts and pages, against the eager
    calls, with eager work between the replays."""
    s = ref.make(50, 3, 21, 28, 4, 128, 16, 30, (300, 10, 77))
    cache, table, starts, _ = ref.on_gpu(s)
    rope = paged.rope_table(30 * 16, 128, device="cuda")
    parents = trees.random_parents(50, 3, 21).cuda()
    q, k, v = (x.cuda() for x in (s.q, s.k, s.v))
    drafts, targets = (torch.randint(0, 2, (3, 21), device="cuda") for _ in range(2))

    def step(cache):
        depths, masks = paged.draft_tree(parents)
        places = starts[:, None] + depths
        turned, _ = paged.append_tokens(cache, table, starts, k, v, q, rope, positions=places)
        out, lse = paged.tree_attention(turned, cache, table, starts, masks, 0.09, return_lse=True)
        return (out, lse, *paged.accept_drafts(cache, table, starts, parents, drafts, targets))

    step(cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(cache)
    for round in range(4):
        gen = torch.Generator().manual_seed(round)
        starts.copy_(torch.tensor([(300, 10, 77), (0, -1, 459), (457, 200, 3), (64, 0, 0)][round]))
        parents.copy_(trees.random_parents(round, 3, 21))
        drafts.copy_(torch.randint(0, 2, (3, 21), generator=gen))
        q.copy_(torch.randn(q.shape, generator=gen))
        pages = torch.randn(s.held[0].shape, generator=gen).to(torch.bfloat16)
        eager = paged.PagedCache(pages.cuda(), pages.cuda() + 1)
        cache.key_pages.copy_(eager.key_pages)
        cache.value_pages.copy_(eager.value_pages)
        torch.cuda.synchronize()
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        for x, y in zip(captured, want):
            assert torch.equal(x, y)
        assert torch.equal(cache.key_pages, eager.key_pages)
        assert torch.equal(cache.value_pages, eager.value_pages)


def test_trees_on_another_stream(gpu):
    """Two calls at once on two streams, each with its own workspace."""
    calls = []
    for seed in (51, 52):
        s = ref.make(seed, 2, 30, 28, 4, 128, 64, 60, (3800, 1000))
        cache, table, starts, _ = ref.on_gpu(s)
        calls.append((s.q.cuda(), cache, table, starts, trees.words(_tree(seed, 2, 30)).cuda(), 0.1))
    want = [paged.tree_attention(*call) for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for _ in range(5):
        for stream, call in zip(streams, calls):
            with torch.cuda.stream(stream):
                got.append(paged.tree_attention(*call))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2])
