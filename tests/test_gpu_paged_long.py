"""Paged attention with values that are not finite, positions without a place and empty rows in the
forms that long contexts take: units shared by workgroups of four waves, partial results joined by
either kernel, two columns' sets in one tile, several column tiles, the products in fp32 away from a
stream's first unit."""

import pytest
import torch

from exp3_amd import paged
from test_gpu_paged import _check_attention
import paged_reference as ref

pytestmark = pytest.mark.gpu

# bits, (query heads, KV heads, head dim), tokens, starts, page size, table width
FORMS = {
    "two column tiles": (16, (12, 2, 128), 3, (2000, 1777, 300), 16, 160),
    "two column tiles, 4 bits": (4, (12, 2, 128), 3, (2000, 1777, 300), 16, 160),
    "d 256": (16, (6, 1, 256), 2, (2500, 901, 1030), 64, 40),
    "d 256, 4 bits": (4, (6, 1, 256), 2, (2500, 901, 1030), 64, 40),
    "a wave per row": (16, (32, 8, 128), 4, tuple(1500 - 61 * b for b in range(8)), 32, 64),
    "a wave per row, 4 bits": (4, (32, 8, 128), 4, tuple(1500 - 61 * b for b in range(8)), 32, 64),
    "a wave per row, d 256, 4 bits": (4, (32, 8, 256), 4, tuple(1500 - 61 * b for b in range(8)), 32, 64),
    "halves": (4, (16, 16, 128), 2, tuple(11998 - 41 * b for b in range(6)), 64, 188),
}


def _make(form, seed, counts=None, starts=None):
    bits, layout, tokens, first, page, width = FORMS[form]
    starts = first if starts is None else starts
    assert width * page > 1024        # up to there a workgroup of eight waves may run a whole stream
    return ref.make(seed, len(starts), tokens, *layout, page, width, starts, counts, bits=bits, spare=2)


def _lengths(s):
    return [int(n) + s.tokens for n in s.starts]


@pytest.mark.parametrize("form", FORMS)
def test_values_that_are_not_finite(gpu, form):
    """Sequence 0: a NaN value and an infinite one in the middle, which every row of KV head 0 sees, and
    an infinite one (4 bits: NaN) at the last token, which the last row sees. Sequence 1: a NaN key at the
    last token. Rows and dims that do not see them are as they were, bit for bit; finite dims of a row that
    sees the last token's value may round another way."""
    s = _make(form, 31)
    want, want_lse = _check_attention(s, 0.1)
    cache, table, starts, _ = ref.on_gpu(s)
    four = s.bits == 4
    group = s.q.shape[2] // s.held[0].shape[1]

    def put(what, b, head, p, d, x):
        page, slot = int(s.table[b, p // s.page]), p % s.page
        if four:
            getattr(cache, what + "_scales")[page, head, slot, d // 32] = 255
        else:
            getattr(cache, what + "_pages")[page, head, slot, d] = float(x)

    lengths, last = _lengths(s), s.tokens - 1
    put("value", 0, 0, lengths[0] // 2, 40, "nan")
    put("value", 0, 0, lengths[0] // 3, 70, "-inf")
    put("value", 0, 0, lengths[0] - 1, 100, "inf")
    put("key", 1, -1, lengths[1] - 1, 3, "nan")
    out, lse = paged.paged_attention(s.q.cuda(), cache, table, starts, 0.1, return_lse=True)
    out, lse = out.double().cpu(), lse.double().cpu()
    bad = torch.zeros_like(out, dtype=torch.bool)
    for d, first in ((40, 0), (70, 0), (100, last)):
        dims = slice(d // 32 * 32, d // 32 * 32 + 32) if four else slice(d, d + 1)
        bad[0, first:, :group, dims] = True
    bad[1, last, -group:] = True
    assert torch.equal(~torch.isfinite(out), bad)
    if not four:
        assert torch.isnan(out[0, :, :group, 40]).all()
        assert (out[0, :, :group, 70] == -float("inf")).all()
        assert (out[0, last, :group, 100] == float("inf")).all()
    assert torch.isnan(out[1, last, -group:]).all()
    sees = torch.zeros_like(bad)
    sees[0, last, :group] = True
    assert torch.equal(out[~bad & ~sees], want[~bad & ~sees])
    torch.testing.assert_close(out[sees & ~bad], want[sees & ~bad], rtol=2.0 ** -7, atol=1e-5)
    nan = torch.zeros_like(lse, dtype=torch.bool)
    nan[1, last, -group:] = True
    assert torch.equal(torch.isnan(lse), nan) and torch.equal(lse[~nan], want_lse[~nan])


@pytest.mark.parametrize("form", FORMS)
def test_values_of_later_tokens(gpu, form):
    """NaN at every new token but the first: the first row is as it was, the others are NaN in the
    dims of KV head 0."""
    s = _make(form, 32)
    want, want_lse = _check_attention(s, 0.1)
    cache, table, starts, _ = ref.on_gpu(s)
    group = s.q.shape[2] // s.held[0].shape[1]
    for b, n in enumerate(_lengths(s)):
        for p in range(n - s.tokens + 1, n):
            page, slot = int(s.table[b, p // s.page]), p % s.page
            if s.bits == 4:
                cache.value_scales[page, 0, slot] = 255
            else:
                cache.value_pages[page, 0, slot] = float("nan")
    out, lse = paged.paged_attention(s.q.cuda(), cache, table, starts, 0.1, return_lse=True)
    out, lse = out.double().cpu(), lse.double().cpu()
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[:, 1:, :group] = True
    assert torch.equal(torch.isnan(out), bad)
    assert torch.equal(out[~bad], want[~bad]) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("form", FORMS)
def test_garbage_behind_the_last_token(gpu, form):
    """Slots behind a sequence's last token and pages of no sequence hold NaN: not seen."""
    s = _make(form, 33)
    want = _check_attention(s, 0.1)
    used = torch.zeros(s.pages, s.page, dtype=torch.bool)
    for b, n in enumerate(_lengths(s)):
        at = torch.arange(n)
        used[s.table[b].long()[at // s.page], at % s.page] = True
    cache, table, starts, _ = ref.on_gpu(s)
    for x in ((cache.key_scales, cache.value_scales) if s.bits == 4 else
              (cache.key_pages, cache.value_pages)):
        x.masked_fill_(~used[:, None, :, None].cuda(), 255 if s.bits == 4 else float("nan"))
    out, lse = paged.paged_attention(s.q.cuda(), cache, table, starts, 0.1, return_lse=True)
    assert torch.equal(out.double().cpu(), want[0]) and torch.equal(lse.double().cpu(), want[1])


@pytest.mark.parametrize("form", FORMS)
def test_places_and_empty_rows(gpu, form):
    """The first sequence a free slot; padding; no live token; a start at the table's end and past it; pages
    outside the cache at the beginning, in the middle, at the end, two units of them, all of them. What
    such pages would hold, and page 0, is NaN."""
    bits, layout, tokens, first, page, width = FORMS[form]
    reach, longest = width * page, first[0]
    starts = (-1, longest, longest - 5, reach - 1, reach, longest - 700, longest - 300, longest - 1)
    counts = (tokens, 1, 0, tokens, tokens, tokens, tokens, tokens)
    s = _make(form, 34, counts, starts)
    s.table[s.table == 0] = s.pages - 1
    s.table[1, 0], s.table[3, -1] = -1, s.pages
    middle = longest // page // 2
    s.table[5, middle:middle + 512 // page] = 2**31 - 1
    s.table[6, middle], s.table[6, middle + 1] = -1, s.pages
    s.table[7, :] = -2**31
    if s.bits == 4:
        for x in s.scales:
            x[0] = 255
        s.held = [ref.values(r, c) for r, c in zip(s.raw, s.scales)]
    else:
        for x in s.held:
            x[0] = float("nan")
    _check_attention(s, 0.1)


@pytest.mark.parametrize("form", FORMS)
def test_keys_of_minus_infinity(gpu, form):
    """bf16: keys of -inf in all but one page, the second sequence's in every page; scores there are -inf
    (dim 0 of the queries is positive). 4 bits have none: NaN scales in pages that no row sees."""
    s = _make(form, 35)
    s.q[..., 0] = 1.0
    if s.bits == 16:
        for page in s.table[0].tolist()[:3] + s.table[0].tolist()[4:] + s.table[1].tolist():
            s.held[0][page, :, :, 0] = -float("inf")
        cache, table, starts, _ = ref.on_gpu(s)
        out, lse = paged.paged_attention(s.q.cuda(), cache, table, starts, 0.1, return_lse=True)
        assert not out[1].any() and torch.equal(lse[1], torch.full_like(lse[1], -float("inf")))
        only = ref.make(36, 1, s.tokens, *FORMS[form][1], s.page, 1, (0,), spare=0)
        only.q, only.table = s.q[:1], s.table[:1, 3:4]
        only.held, only.pages = s.held, s.pages
        only.starts = torch.tensor([s.page - 1], dtype=torch.int32)
        for i in range(s.tokens):                 # each row by itself: it sees that one page
            only.q, only.tokens = s.q[:1, i:i + 1], 1
            want, want_lse, off, lse_off = ref.attention(only, 0.1)
            got = out[:1, i:i + 1].double().cpu()
            assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + off).all()
            assert ((lse[:1, i:i + 1].double().cpu() - want_lse).abs() <= lse_off).all()
    else:
        s.table[1, 5:] = -1
        unseen = sorted(set(range(s.pages)) - set(s.table.flatten().tolist()))
        for x in s.scales:
            x[unseen] = 255
        s.held = [ref.values(r, c) for r, c in zip(s.raw, s.scales)]
        _check_attention(s, 0.1)
