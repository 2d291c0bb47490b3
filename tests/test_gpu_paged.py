"""The paged KV cache on the GPU against its definition in 64 bits: append with rotation, read
back, attention; bf16 and 4-bit pages, head dims 128 and 256, page sizes from 16 to 1024, free
slots, padding, positions without a place, strided inputs, special values, captured graphs.

4-bit contents are compared for equality (the kernel rounds the exact value). bf16 rows: two
fp32 products and their sum, then one rounding: |got - want| <= 2^-8 |want| + 2^-22 (|a| + |b|).
Attention: the bounds that paged_reference.attention derives, and the output's half step."""

import pytest
import torch

from exp3_amd import attention, paged
import paged_reference as ref

pytestmark = pytest.mark.gpu

LAYOUTS = ((28, 4, 128), (16, 4, 256), (8, 8, 128), (20, 1, 128), (34, 2, 256))


def _bf16_close(got, want, scale=8.0):
    """scale: above the largest |a| + |b| of the inputs."""
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    off = (got - want).abs() - 2.0 ** -8 * want.abs()
    assert off.max() <= 2.0 ** -22 * scale, off.max().item()


def _check_append(s, rope=True, interleaved=False, q=True, keys=True):
    cache, table, starts, counts = ref.on_gpu(s)
    got_q, got_k = paged.append_tokens(
        cache, table, starts, s.k.cuda(), s.v.cuda(), s.q.cuda() if q else None,
        tuple(t.cuda() for t in s.rope) if rope else None, counts, interleaved, keys)
    want_q, want_k, want_key, want_value = ref.append(s, rope, interleaved)
    assert (got_q is None) == (not q) and (got_k is None) == (not keys)
    if q:
        _bf16_close(got_q, want_q)
    if keys:
        _bf16_close(got_k, want_k)
    key, value = ref.contents(cache)
    if s.bits == 4:
        assert torch.equal(key, want_key)
    else:
        _bf16_close(key, want_key)
        untouched = want_key == s.held[0].double()
        assert torch.equal(key[untouched], want_key[untouched])
    assert torch.equal(value, want_value)
    return cache


def _check_attention(s, scale, max_keys=None, q=None):
    cache, table, starts, counts = ref.on_gpu(s)
    out, lse = paged.paged_attention(s.q.cuda() if q is None else q, cache, table, starts, scale,
                                     counts, max_keys, return_lse=True)
    want, want_lse, out_off, lse_off = ref.attention(s, scale)
    out, lse = out.double().cpu(), lse.double().cpu()
    empty = torch.isinf(want_lse)
    assert (out[empty] == 0).all() and torch.equal(lse[empty], want_lse[empty])
    assert torch.isfinite(out).all()
    off = (out - want).abs() - 2.0 ** -8 * want.abs() - out_off
    assert off.max() <= 0, (off.max().item(), out_off.max().item())
    off = (lse - want_lse).abs()[~empty] - lse_off[~empty]
    assert off.numel() == 0 or off.max() <= 0, off.max().item()
    return out, lse


# ------------------------------------------------------------------- append

@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("page", (16, 64, 1024))
@pytest.mark.parametrize("layout", LAYOUTS)
def test_append_tokens(gpu, layout, page, bits):
    width = 2 if page > 64 else 5
    s = ref.make(1, 3, 9, *layout, page, width, (0, page - 4, 3), bits=bits)
    _check_append(s)


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("dim,rotary", ((128, 16), (128, 96), (128, 112), (256, 64), (256, 256)))
@pytest.mark.parametrize("interleaved", (False, True))
def test_append_rotations(gpu, dim, rotary, interleaved, bits):
    s = ref.make(2, 2, 5, 6, 2, dim, 32, 3, (40, 1), bits=bits, rotary=rotary)
    _check_append(s, interleaved=interleaved)


@pytest.mark.parametrize("bits", (16, 4))
def test_append_parts(gpu, bits):
    s = ref.make(3, 2, 3, 4, 2, 128, 16, 4, (0, 17), bits=bits)
    _check_append(s, rope=False)
    _check_append(s, q=False)
    _check_append(s, q=False, keys=False)


@pytest.mark.parametrize("bits", (16, 4))
def test_append_free_slots_padding_and_reach(gpu, bits):
    """A free slot, padding, no tokens at all, the end of the table, page ids outside the cache,
    and starts next to 2^31: nothing of the other slots changes."""
    s = ref.make(4, 8, 6, 4, 2, 128, 16, 3, (-1, 5, 20, 45, 0, 14, 2**31 - 3, -2**31),
                 counts=(6, 3, 0, 6, -4, 9, 6, 6), bits=bits)
    s.table[5, 1] = -1
    s.table[1, 0] = s.pages
    s.table[4, :] = 2**31 - 1
    _check_append(s)


def test_append_far_positions(gpu):
    """Rotation and rows behind position 131000, where an angle in fp32 would be off by 2^-8."""
    s = ref.make(5, 1, 40, 4, 2, 128, 1024, 129, (131072 - 20,), bits=4, spare=0)
    _check_append(s)


def test_append_strided_inputs(gpu):
    s = ref.make(6, 2, 7, 6, 2, 128, 16, 3, (3, 0), bits=16)
    want = _check_append(s)
    fused = torch.cat((s.q, s.k, s.v), 2).cuda()
    q, k, v = fused.split((6, 2, 2), 2)
    cache, table, starts, _ = ref.on_gpu(s)
    wide = torch.full((2, 8), -7, dtype=torch.int32, device="cuda")
    wide[:, 1:4] = table
    rope = tuple(t.cuda() for t in s.rope)
    paged.append_tokens(cache, wide[:, 1:4], starts, k, v, q, rope)
    assert torch.equal(cache.key_pages, want.key_pages)
    assert torch.equal(cache.value_pages, want.value_pages)
    # a layout that is copied first: odd row starts, a transposed view, a lazy negation
    odd = torch.zeros(2, 7, 2, 129, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(k)
    turned = v.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    again = ref.on_gpu(s)[0]
    paged.append_tokens(again, table, starts, odd, torch._neg_view(-turned), rope=rope)
    assert torch.equal(again.key_pages, want.key_pages)
    assert torch.equal(again.value_pages, want.value_pages)


def test_append_4bit_borders_and_special_values(gpu):
    """Unrotated rows at every border of the grid and next to it, largest values around
    the scale's step, zeros, subnormals, huge values, infinities and NaN."""
    s = ref.make(7, 1, 16, 2, 2, 128, 16, 1, (0,), bits=4)
    grid = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, -5])
    step = 2.0 ** torch.arange(-8, 8).float()
    rows = (grid.repeat(8)[None] * step[:, None])[:, None].repeat(1, 2, 1)
    rows[:, 1] *= 1 + 2.0 ** -7                       # one bf16 step further
    rows[3, :, 32:64] = 0
    rows[4, 0, 0], rows[4, 1, 0] = 3.49, 3.51
    rows[5] *= 2.0 ** -130
    rows[6, 0, 33], rows[6, 1, 70] = float("inf"), float("nan")
    rows[7] = 3.3e38
    rows[8] = -1e-40
    rows[9, 0, 5], rows[9, 1, 5] = 7 * step[9], 6.9375 * step[9]
    s.k = rows[None].to(torch.bfloat16)
    s.v = -s.k
    cache, table, starts, _ = ref.on_gpu(s)
    paged.append_tokens(cache, table, starts, s.k.cuda(), s.v.cuda())
    _, _, want_key, want_value = ref.append(s, rope=False)
    for got, want in zip(ref.contents(cache), (want_key, want_value)):
        torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
    assert torch.isnan(ref.contents(cache)[0]).sum() == 64


def test_append_4bit_rotated_borders(gpu):
    """Rotated values next to a border: rotations by exact angles leave them on it."""
    s = ref.make(8, 1, 4, 2, 2, 128, 16, 1, (0,), bits=4)
    s.rope = (torch.tensor([1.0, 0.5, 1 + 2.0 ** -23, 1 - 2.0 ** -24]).repeat(4)[:, None].repeat(1, 64),
              torch.tensor([0.0, 2.0 ** -30, -2.0 ** -30, 2.0 ** -24]).repeat(4)[:, None].repeat(1, 64))
    grid = torch.tensor([6, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, -5])
    s.k = grid.repeat(8)[None, None, None].repeat(1, 4, 2, 1).to(torch.bfloat16)
    _check_append(s)


# ------------------------------------------------------------------- gather

@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("layout,page", (((28, 4, 128), 16), ((16, 4, 256), 128), ((3, 3, 128), 32)))
def test_gather_tokens(gpu, layout, page, bits):
    s = ref.make(9, 6, 37, *layout, page, 4, (0, 5, -1, 4 * page - 30, 2, 9),
                 counts=(37, 11, 37, 37, 0, 37), bits=bits)
    s.table[5, 0], s.table[1, 0] = -3, s.pages
    cache, table, starts, counts = ref.on_gpu(s)
    for got, want in zip(paged.gather_tokens(cache, table, starts, 37, counts), ref.gather(s)):
        assert got.dtype == torch.bfloat16 and torch.equal(got.double().cpu(), want)
    whole = paged.gather_tokens(cache, table, torch.zeros_like(starts), 37)
    s.starts, s.counts = torch.zeros_like(s.starts), None
    for got, want in zip(whole, ref.gather(s)):
        assert torch.equal(got.double().cpu(), want)


def test_gather_4bit_nan_scale(gpu):
    s = ref.make(10, 1, 16, 2, 2, 128, 16, 1, (0,), bits=4, spare=0)
    s.scales[0][0, 1, 3, 2] = 255
    s.scales[1][0, 0, 5, 0] = 2
    s.held = [ref.values(r, c) for r, c in zip(s.raw, s.scales)]
    cache, table, starts, _ = ref.on_gpu(s)
    for got, want in zip(paged.gather_tokens(cache, table, starts, 16), ref.gather(s)):
        torch.testing.assert_close(got.double().cpu(), want, rtol=0, atol=0, equal_nan=True)


# ---------------------------------------------------------------- attention

LENGTHS = (1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 256, 257, 300, 511, 513, 767)


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("tokens", (1, 3))
def test_attention_lengths(gpu, layout, tokens, bits):
    """One batch with a sequence of every length, and a free slot."""
    starts = tuple(n - tokens for n in LENGTHS if n >= tokens) + (-1,)
    s = ref.make(11, len(starts), tokens, *layout, 16, 48, starts, bits=bits, sharp=2.0, spare=0)
    _check_attention(s, layout[2] ** -0.5)


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("page", (32, 128, 1024))
def test_attention_pages(gpu, page, bits):
    s = ref.make(12, 3, 2, 28, 4, 128, page, -(-1500 // page), (1498, 77, 1023), bits=bits)
    _check_attention(s, 0.1)
    _check_attention(s, 0.1, max_keys=1500)
    _check_attention(s, 0.1, max_keys=1)          # a wrong bound costs time, not results


# more keys than workgroups x steps, few and many streams
@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("batch,layout,keys,tokens", ((1, (4, 2, 128), 70001, 1),
                                                      (1, (2, 1, 256), 40003, 2),
                                                      (40, (8, 8, 128), 1900, 1),
                                                      (6, (16, 16, 128), 12000, 2),
                                                      (5, (24, 3, 128), 66000, 1)))
def test_attention_long_and_wide(gpu, batch, layout, keys, tokens, bits):
    starts = tuple(max(0, keys - tokens - 41 * b) for b in range(batch))
    s = ref.make(13, batch, tokens, *layout, 64, -(-keys // 64), starts, bits=bits, sharp=4.0,
                 spare=0)
    _check_attention(s, layout[2] ** -0.5)


@pytest.mark.parametrize("tokens,layout", ((8, (28, 4, 128)), (16, (16, 4, 256)), (33, (8, 8, 128)),
                                           (5, (40, 2, 128))))
@pytest.mark.parametrize("bits", (16, 4))
def test_attention_many_tokens(gpu, tokens, layout, bits):
    """More rows than one matrix tile; the first tokens of a sequence see only themselves."""
    s = ref.make(14, 4, tokens, *layout, 32, 20, (0, 1, 130, 600), bits=bits)
    _check_attention(s, 0.09)


@pytest.mark.parametrize("bits", (16, 4))
def test_attention_empty_rows(gpu, bits):
    """Free slots, padding, positions past the table, pages outside the cache (one in the middle,
    all of a sequence), starts next to 2^31."""
    s = ref.make(15, 9, 4, 14, 2, 128, 16, 20, (-1, 100, 250, 318, 77, 50, 2**31 - 2, -9, 0),
                 counts=(4, 2, 0, 4, 4, 4, 4, 4, -1), bits=bits)
    s.table[1, 3], s.table[4, :], s.table[5, 3] = -1, 2**31 - 1, s.pages
    _check_attention(s, 0.1)


@pytest.mark.parametrize("bits", (16, 4))
def test_attention_more_sequences_than_lanes(gpu, bits):
    """The units of 150 sequences, free slots and padding among them, are found over three scans."""
    starts = tuple(-1 if b % 7 == 3 else 37 * b % 1900 for b in range(150))
    counts = tuple(b % 4 for b in range(150))
    s = ref.make(24, 150, 3, 6, 3, 128, 128, 15, starts, counts, bits=bits, spare=0)
    _check_attention(s, 0.1)


@pytest.mark.parametrize("bits", (16, 4))
def test_attention_of_66000_sequences(gpu, bits):
    """More sequences than a grid has rows, in both forms (eight waves per stream; shared units),
    and as many appended and read back: every fifth one is the same."""
    s = ref.make(25, 5, 1, 2, 1, 128, 64, 10, (600, 0, -1, 63, 311), bits=bits)
    want, want_lse, off, lse_off = (x.cuda() for x in ref.attention(s, 0.1))
    cache, table, starts, _ = ref.on_gpu(s)
    many = [x.repeat(13200, *([1] * (x.dim() - 1))) for x in (s.q.cuda(), table, starts)]
    for bound in (None, 601):
        out, lse = paged.paged_attention(many[0], cache, *many[1:], 0.1, max_keys=bound,
                                         return_lse=True)
        out, lse = out.view(13200, 5, 1, 2, 128).double(), lse.view(13200, 5, 1, 2).double()
        assert ((out - want).abs() <= 2.0 ** -8 * want.abs() + off).all()
        assert ((lse == want_lse) | ((lse - want_lse).abs() <= lse_off)).all()
    k, _ = paged.gather_tokens(cache, many[1], many[2], 1)
    few, _ = paged.gather_tokens(cache, table, starts, 1)
    assert (k.view(13200, *few.shape) == few).all()
    q, k = paged.append_tokens(cache, many[1], torch.full_like(many[2], -1), k, k, many[0],
                               return_keys=True)
    assert not q.any() and not k.any()


@pytest.mark.parametrize("bits", (16, 4))
def test_attention_of_a_long_chunk(gpu, bits):
    """Many column tiles of one stream, each with keys of its own."""
    s = ref.make(26, 2, 150, 7, 1, 128, 32, 10, (0, 130), (150, 77), bits=bits)
    _check_attention(s, 0.1)


@pytest.mark.parametrize("bits", (16, 4))
def test_pages_past_32_bit_offsets(gpu, bits):
    """The same tokens in the first and in the last pages of a cache of more than 4 GiB an array."""
    pages = 20000 if bits == 16 else 76000
    cache = paged.empty_pages(pages, 128, 8, 128, "cuda", four_bit=bits == 4)
    assert cache.key_pages.numel() * cache.key_pages.element_size() > 1 << 32
    gen = torch.Generator("cuda").manual_seed(5)
    q, k, v = (torch.randn(1, 700, h, 128, generator=gen, device="cuda").to(torch.bfloat16)
               for h in (16, 8, 8))
    start = torch.zeros(1, dtype=torch.int32, device="cuda")
    rope = paged.rope_table(768, 128, device="cuda")
    seen = []
    for first in (0, pages - 6):
        table = torch.arange(first, first + 6, dtype=torch.int32, device="cuda")[None]
        turned, _ = paged.append_tokens(cache, table, start, k, v, q, rope)
        held = paged.gather_tokens(cache, table, start, 700)
        out = paged.paged_attention(turned[:, -1:].contiguous(), cache, table, start + 699, 0.1)
        seen.append((turned, *held, out))
    assert all(torch.equal(a, b) for a, b in zip(*seen))
    if bits == 16:
        assert torch.equal(seen[0][2], v)
    # the last pages were written, not the first ones again
    cache.key_pages[:6] = 0
    cache.value_pages[:6] = 0
    assert torch.equal(paged.gather_tokens(cache, table, start, 700)[1], seen[0][2])


@pytest.mark.parametrize("scale", (-0.2, 0.0, 3.0))
@pytest.mark.parametrize("bits", (16, 4))
def test_attention_scales(gpu, scale, bits):
    s = ref.make(16, 2, 1, 28, 4, 128, 64, 11, (699, 20), bits=bits)
    _check_attention(s, scale)


@pytest.mark.parametrize("bits", (16, 4))
def test_attention_garbage_behind_the_last_token(gpu, bits):
    """Slots behind a sequence's last token and pages of no sequence hold NaN: not seen."""
    s = ref.make(17, 3, 1, 12, 2, 128, 32, 9, (5, 130, 256), bits=bits)
    want = _check_attention(s, 0.1)
    used = torch.zeros(s.pages, s.page, dtype=torch.bool)
    for b in range(3):
        for p in range(int(s.starts[b]) + 1):
            used[int(s.table[b, p // 32]), p % 32] = True
    cache, table, starts, _ = ref.on_gpu(s)
    for x in ((cache.key_scales, cache.value_scales) if bits == 4 else
              (cache.key_pages, cache.value_pages)):
        x.masked_fill_(~used[:, None, :, None].cuda(), 255 if bits == 4 else float("nan"))
    out, lse = paged.paged_attention(s.q.cuda(), cache, table, starts, 0.1, return_lse=True)
    assert torch.equal(out.double().cpu(), want[0]) and torch.equal(lse.double().cpu(), want[1])


@pytest.mark.parametrize("bits", (16, 4))
def test_attention_special_values(gpu, bits):
    """A NaN key makes the rows of its heads NaN where they see it, and no others; a NaN value
    reaches its dims only."""
    s = ref.make(18, 2, 2, 12, 2, 128, 16, 20, (300, 299), bits=bits)
    want, _ = _check_attention(s, 0.1)
    cache, table, starts, _ = ref.on_gpu(s)

    def put(b, head, p, keys, values):
        page, slot = int(s.table[b, p // 16]), p % 16
        if bits == 4:      # a NaN scale is NaN for its 32 dims
            if keys:
                cache.key_scales[page, head, slot, 1] = 255
            if values:
                cache.value_scales[page, head, slot, 1] = 255
        else:
            if keys:
                cache.key_pages[page, head, slot, 40] = float("nan")
            if values:
                cache.value_pages[page, head, slot, 40] = float("nan")

    put(0, 1, 301, True, False)         # seen by the second token of sequence 0 only
    put(1, 0, 7, False, True)
    out = paged.paged_attention(s.q.cuda(), cache, table, starts, 0.1).double().cpu()
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 1, 6:] = True
    bad[1, :, :6, 32:64 if bits == 4 else 41] = True
    if bits == 16:
        bad[1, :, :6, 32:40] = False
    assert torch.equal(torch.isnan(out), bad)
    assert torch.equal(out[~bad], want[~bad])


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("layout", ((12, 2, 128), (6, 1, 256)))
def test_attention_special_values_of_later_tokens(gpu, layout, bits):
    """Values that are not finite at tokens that only some of the rows see: the others are as
    they were, bit for bit, and those that see them are NaN or infinite."""
    s = ref.make(23, 2, 5, *layout, 16, 20, (200, 61), bits=bits)
    want, _ = _check_attention(s, 0.1)
    cache, table, starts, _ = ref.on_gpu(s)
    for b, p, dim, x in ((0, 202, 40, "nan"), (0, 204, 100, "inf"), (1, 65, 7, "-inf")):
        page, slot = int(s.table[b, p // 16]), p % 16
        if bits == 4:
            cache.value_scales[page, 0, slot, dim // 32] = 255
        else:
            cache.value_pages[page, 0, slot, dim] = float(x)
    out = paged.paged_attention(s.q.cuda(), cache, table, starts, 0.1).double().cpu()
    off = torch.zeros_like(out, dtype=torch.bool)
    heads = layout[0] // layout[1]
    for b, first, dim in ((0, 2, 40), (0, 4, 100), (1, 4, 7)):
        dims = slice(dim // 32 * 32, dim // 32 * 32 + 32) if bits == 4 else slice(dim, dim + 1)
        off[b, first:, :heads, dims] = True
    assert torch.equal(~torch.isfinite(out), off)
    # rounding of the rows that see them goes another way in their finite dims
    torch.testing.assert_close(out[~off], want[~off], rtol=2.0 ** -7, atol=1e-4)
    assert torch.equal(out[0, :2], want[0, :2]) and torch.equal(out[1, :4], want[1, :4])
    if bits == 16:
        assert (out[0, 4, :heads, 100] == float("inf")).all()
        assert (out[1, 4, :heads, 7] == -float("inf")).all()


def test_attention_one_sided_scores(gpu):
    """Scores far from 0 on either side: the maximum is subtracted."""
    s = ref.make(19, 1, 1, 4, 2, 128, 64, 12, (700,))
    s.held[0][:] = 3.0
    s.q[:] = 2.0
    for scale in (4.0, -4.0):
        _check_attention(s, scale)


@pytest.mark.parametrize("bits", (16, 4))
def test_attention_strided_queries_and_repeats(gpu, bits):
    s = ref.make(20, 3, 2, 28, 4, 128, 16, 30, (400, 12, 250), bits=bits)
    want = _check_attention(s, 0.1)
    fused = torch.zeros(3, 2, 36, 128, dtype=torch.bfloat16, device="cuda")
    fused[:, :, :28] = s.q.cuda()
    for q in (fused[:, :, :28], s.q.cuda().transpose(1, 2).contiguous().transpose(1, 2)):
        got = _check_attention(s, 0.1, q=q)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ----------------------------------------------------------- as they are used

def _step(cache, table, starts, fused, rope, scale, heads):
    q, k, v = fused.split(heads, 2)
    q, _ = paged.append_tokens(cache, table, starts, k, v, q, rope)
    return q, paged.paged_attention(q, cache, table, starts, scale)


@pytest.mark.parametrize("bits", (16, 4))
def test_prompt_then_steps(gpu, bits):
    """A prompt appended, prefilled by the backend on the returned Q and K, then decode steps
    through the cache: each output against attention in 64 bits over all tokens so far (a
    4-bit cache: over the values that it holds)."""
    heads, dim, prompt, steps, scale = (28, 4, 4), 128, 300, 5, 128 ** -0.5
    gen = torch.Generator("cuda").manual_seed(3)
    fused = torch.randn(1, prompt + steps, 36, dim, generator=gen, device="cuda").to(torch.bfloat16)
    cache = paged.empty_pages(30, 16, 4, dim, "cuda", four_bit=bits == 4)
    table = torch.randperm(30, generator=gen, device="cuda")[None, :20].int()
    rope = paged.rope_table(320, dim, device="cuda")
    start = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, k, v = fused[:, :prompt].split(heads, 2)
    q, k = paged.append_tokens(cache, table, start, k, v, q, rope, return_keys=True)
    backend = attention.AttentionBackend(register=False, dense_impl="hip")

    class Layer:
        layer_idx = 0

    first, _ = backend.forward(Layer(), q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2),
                               None, scale)
    if bits == 16:
        # the whole prompt through the cache: the prefill rounds its probabilities to bf16 (an
        # output by 2^-8 of the largest value), both round their output
        again = paged.paged_attention(q, cache, table, start, scale)
        torch.testing.assert_close(again.float(), first.float(), rtol=2.0 ** -7,
                                   atol=2.0 ** -8 * v.abs().max().item())
    for i in range(prompt, prompt + steps):
        q, out = _step(cache, table, start + i, fused[:, i:i + 1], rope, scale, heads)
        _bf16_close(q[0, 0], ref.rotated(fused[0, i, :28].double().cpu(),
                                         *(t[i].double().cpu() for t in rope)))
        held = paged.gather_tokens(cache, table, start, i + 1)
        s = ref.make(0, 1, 1, 28, 4, dim, 512, 1, (i,), spare=0)
        s.q, s.table[:] = q.cpu(), 0
        s.held = [torch.zeros(1, 4, 512, dim, dtype=torch.float64) for _ in range(2)]
        for x, rows in zip(s.held, held):
            x[0, :, :i + 1] = rows[0].double().cpu().transpose(0, 1)
        want, _, off, _ = ref.attention(s, scale)
        assert ((out.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + off).all()
    # what the cache holds of the prompt is what was appended
    key, value = paged.gather_tokens(cache, table, start, prompt)
    if bits == 16:
        assert torch.equal(key, k) and torch.equal(value, v)
    else:
        assert torch.equal(value.double().cpu(), ref.four_bit(v.double().cpu()))


def test_captured_steps_with_other_lengths(gpu):
    """A captured append and attention, replayed with other lengths and tables, eager work and
    other graphs between the replays."""
    heads, scale = (12, 2, 2), 0.1
    gen = torch.Generator("cuda").manual_seed(4)
    rope = paged.rope_table(64 * 16, 128, device="cuda")
    fused = torch.randn(4, 1, 16, 128, generator=gen, device="cuda").to(torch.bfloat16)

    def fresh(bits):
        s = ref.make(21, 4, 1, 12, 2, 128, 16, 64, (0, 0, 0, 0), bits=bits)
        return ref.on_gpu(s)

    graphs = []
    for bits in (16, 4):
        cache, table, starts, _ = fresh(bits)
        _step(cache, table, starts, fused, rope, scale, heads)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _, out = _step(cache, table, starts, fused, rope, scale, heads)
        graphs.append((bits, graph, cache, table, starts, out))
    for lengths in ((5, 900, -1, 1023), (1023, 0, 300, 255), (0, 0, -5, 0), (700, 701, 702, 703)):
        fused.copy_(torch.randn(4, 1, 16, 128, generator=gen, device="cuda"))
        now = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        for bits, graph, cache, table, starts, out in graphs:
            eager = paged.PagedCache(*(x if x is None else x.clone() for x in (
                cache.key_pages, cache.value_pages, cache.key_scales, cache.value_scales)))
            starts.copy_(now)
            _, want = _step(eager, table, now, fused, rope, scale, heads)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            assert torch.equal(cache.key_pages, eager.key_pages)


def test_two_streams(gpu):
    s = ref.make(22, 2, 1, 28, 4, 128, 64, 80, (5000, 4000), bits=4, spare=0)
    cache, table, starts, _ = ref.on_gpu(s)
    q = s.q.cuda()
    want = paged.paged_attention(q, cache, table, starts, 0.1)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(4):
        for stream, got in zip(streams, outs):
            with torch.cuda.stream(stream):
                got.append(paged.paged_attention(q, cache, table, starts, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for got in outs for x in got)


def test_empty_calls_and_refusals(gpu):
    cache = paged.empty_pages(8, 16, 2, 128, "cuda")
    table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    starts = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.zeros(1, 0, 2, 128, dtype=torch.bfloat16, device="cuda")
    q, k = paged.append_tokens(cache, table, starts, x, x, x, return_keys=True)
    assert q.shape == k.shape == x.shape
    assert paged.gather_tokens(cache, table, starts, 0)[0].shape == (1, 0, 2, 128)
    assert paged.paged_attention(x, cache, table, starts, 0.1).shape == x.shape
    assert paged.gather_tokens(cache, table[:0], starts[:0], 3)[0].shape == (0, 3, 2, 128)
    x = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16, device="cuda")
    short = paged.rope_table(63, 128, device="cuda")
    for call in (lambda: paged.append_tokens(cache, table, starts, x, x, rope=short),
                 lambda: paged.append_tokens(cache, table, starts, x, x[..., :64]),
                 lambda: paged.append_tokens(cache, table, starts, x[:, :, :1], x[:, :, :1]),
                 lambda: paged.append_tokens(cache, table, starts, x.half(), x.half()),
                 lambda: paged.append_tokens(cache, table, starts.cpu(), x, x),
                 lambda: paged.append_tokens(cache, table, starts, x, x, x.repeat(1, 2, 1, 1)),
                 lambda: paged.append_tokens(cache, table, starts, x, x,
                                             rope=tuple(t.double() for t in short)),
                 lambda: paged.gather_tokens(cache, table, starts, -1),
                 lambda: paged.paged_attention(x.repeat(1, 1, 2, 1)[:, :, :3], cache, table, starts,
                                               0.1),
                 lambda: paged.paged_attention(x, cache, table.long(), starts, 0.1),
                 lambda: paged.paged_attention(x, cache, table, starts, 0.1, max_keys=-1),
                 lambda: paged.paged_attention(x.float(), cache, table, starts, 0.1)):
        with pytest.raises(ValueError):
            call()


def test_tensors_that_require_a_gradient(gpu):
    """Refused while gradients are recorded, taken otherwise."""
    cache = paged.empty_pages(8, 16, 2, 128, "cuda")
    table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    starts = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.ones(1, 1, 2, 128, dtype=torch.bfloat16, device="cuda")
    leaf = torch.ones_like(x).requires_grad_()
    for call in (lambda y: paged.append_tokens(cache, table, starts, y, x),
                 lambda y: paged.append_tokens(cache, table, starts, x, y),
                 lambda y: paged.append_tokens(cache, table, starts, x, x, y),
                 lambda y: paged.paged_attention(y, cache, table, starts, 0.1)):
        for y in (leaf, leaf * 2):
            with pytest.raises(ValueError, match="requires a gradient"):
                call(y)
        for off in (torch.no_grad, torch.inference_mode):
            with off():
                call(leaf)
                call(leaf * 2)
        assert call(leaf.detach()) is not None


@pytest.mark.parametrize("bits", (16, 4))
def test_sequences_with_a_common_prefix(gpu, bits):
    """Pages that several sequences read, each with pages of its own behind them."""
    s = ref.make(23, 3, 1, 8, 2, 128, 16, 20, (200, 150, 319), bits=bits)
    s.table[1:, :9] = s.table[0, :9]
    cache, table, starts, _ = ref.on_gpu(s)
    want, want_lse, off, lse_off = ref.attention(s, 0.1)
    got, lse = paged.paged_attention(s.q.cuda(), cache, table, starts, 0.1, return_lse=True)
    assert ((got.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + off).all()
    assert ((lse.double().cpu() - want_lse).abs() <= lse_off).all()


@pytest.mark.parametrize("keys", (40, 700, 5000))
def test_rows_without_a_score_above_minus_infinity(gpu, keys):
    """Keys of -inf: such a row gives 0 and -inf where all its scores are -inf, and counts the
    finite ones alone where some are."""
    s = ref.make(24, 2, 1, 4, 2, 128, 16, keys // 16 + 1, (keys - 1, keys - 1), spare=0)
    for page in s.table[0].tolist():
        s.held[0][page, :, :, 0] = -float("inf")
    mixed = s.table[1].tolist()
    for page in mixed[1:]:
        s.held[0][page, :, :, 0] = -float("inf")
    s.q[..., 0] = 1.0
    cache, table, starts, _ = ref.on_gpu(s)
    got, lse = paged.paged_attention(s.q.cuda(), cache, table, starts, 0.1, return_lse=True)
    assert not got[0].any() and torch.equal(lse[0], torch.full_like(lse[0], -float("inf")))
    alone, alone_lse = paged.paged_attention(s.q[1:].cuda(), cache, table[1:], starts[1:] * 0 + 15,
                                             0.1, return_lse=True)
    # the same 16 keys, joined with empty parts: both round to bf16, and weights of 1 are exact
    assert torch.equal(got[1:], alone) and torch.equal(lse[1:], alone_lse)


def test_graphs_that_share_a_pool(gpu):
    """Two captured calls whose workspaces may be the same memory, replayed in turn."""
    calls = []
    for seed, bits, lengths in ((25, 16, (3000, 900)), (26, 4, (700, 5100))):
        s = ref.make(seed, 2, 1, 28, 4, 128, 64, 80, lengths, bits=bits, spare=0)
        cache, table, starts, _ = ref.on_gpu(s)
        calls.append((s.q.cuda(), cache, table, starts, 0.1))
    want = [paged.paged_attention(*call) for call in calls]
    torch.cuda.synchronize()
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for call in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = paged.paged_attention(*call)
        graphs.append((graph, out))
    for _ in range(3):
        for (graph, out), expected in zip(graphs, want):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, expected)
        assert torch.equal(paged.paged_attention(*calls[0]), want[0])


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("layout", ((28, 4, 128), (16, 4, 256)))
def test_calls_larger_than_the_caches(gpu, layout, bits):
    """One call of 400 MB and more, with padding, against calls of a few tokens each."""
    q_heads, kv_heads, dim = layout
    heads, total, part, live = (q_heads, kv_heads, kv_heads), 28000, 875, 27001
    gen = torch.Generator("cuda").manual_seed(27)
    x = torch.randn(1, total, sum(heads), dim, generator=gen, device="cuda").to(torch.bfloat16)
    rope = paged.rope_table(28032, dim // 2, device="cuda")
    table = torch.randperm(500, generator=gen, device="cuda")[None, :438].int()
    start, count = (torch.tensor([n], dtype=torch.int32, device="cuda") for n in (3, live))
    one, many = (paged.PagedCache(*(None if t is None else t.zero_() for t in (
        c.key_pages, c.value_pages, c.key_scales, c.value_scales))) for c in (
            paged.empty_pages(500, 64, kv_heads, dim, "cuda", four_bit=bits == 4) for _ in range(2)))
    q, k = paged.append_tokens(one, table, start, *x.split(heads, 2)[1:], x[:, :, :q_heads], rope,
                               count, return_keys=True)
    for at in range(0, total, part):
        few = x[:, at:at + part].split(heads, 2)
        few_q, few_k = paged.append_tokens(many, table, start + at, *few[1:], few[0], rope,
                                           count - at, return_keys=True)
        assert torch.equal(q[:, at:at + part], few_q) and torch.equal(k[:, at:at + part], few_k)
    assert not q[:, live:].any() and not k[:, live:].any() and q[:, :live].any()
    assert torch.equal(one.key_pages, many.key_pages)
    assert torch.equal(one.value_pages, many.value_pages)
    if bits == 4:
        assert torch.equal(one.key_scales, many.key_scales)
        assert torch.equal(one.value_scales, many.value_scales)
    # read back in one call of as many bytes
    times = 8
    rows, starts = table.repeat(times, 1), start.repeat(times)
    whole = paged.gather_tokens(one, rows, starts, total, count.repeat(times))
    for at in range(0, total, part):
        few = paged.gather_tokens(one, table, start + at, part, count - at)
        for got, want in zip(whole, few):
            assert torch.equal(got[:, at:at + part], want.expand(times, -1, -1, -1))


def test_append_for_66000_sequences(gpu):
    """More sequences than a grid has rows, each with a page of its own: what is read back is what
    was appended."""
    batch = 66000
    gen = torch.Generator("cuda").manual_seed(28)
    cache = paged.empty_pages(batch, 16, 1, 128, "cuda")
    table = torch.randperm(batch, generator=gen, device="cuda")[:, None].int()
    starts = torch.arange(batch, dtype=torch.int32, device="cuda") % 17 - 1      # some free
    k, v = (torch.randn(batch, 1, 1, 128, generator=gen, device="cuda").to(torch.bfloat16)
            for _ in range(2))
    _, rotated = paged.append_tokens(cache, table, starts, k, v, return_keys=True)
    live = (starts >= 0)[:, None, None, None]
    assert torch.equal(rotated, k * live)
    key, value = paged.gather_tokens(cache, table, starts, 1)
    assert torch.equal(key, k * live) and torch.equal(value, v * live)
