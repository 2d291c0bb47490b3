"""Gathered weights where nothing but the roundings of scale and LSE is off: scores of whole numbers,
exact in fp32, near 37000, whose LSE in base 2 is near 9200.

A kernel that takes 2^(s' x - L') for 2^(s x - L), s' and L' rounded, is off by up to 9200 (2^-24 +
2^-24) ln 2 = 7.6e-4 of a weight; here a weight is held to some 2^-20. With t = s x - L that is: 2^-24
|t| ln 2 each for the rounding of s' x - L' and for taking s' x for L' in the correction, 2^-22 each for
the exponentials of the weight and of the correction, 2^-30 for the correction's own roundings, and
(c + 16) 2^-24 for the sums of c columns, one after the other, of lanes and of workgroups."""

import math

import pytest
import torch

from exp3_amd import paged

LARGE = 96                                    # four such dims: 36864
# scales of 32 bits whose product with log2 e rounds by nearly half a step, down and up
SCALES = (0.17353136837482452, 0.17352473735809326)
START = 500


def _inputs(heads, kv, dim, tokens, scale):
    """q, keys [N, Hkv, D] and LSEs; the sum, its bound, and s x - L and visibility of all rows."""
    gen = torch.Generator().manual_seed(heads + tokens + dim)
    q = torch.randint(0, 2, (tokens, heads, dim), generator=gen).double() * 2 - 1
    k = torch.randint(0, 2, (START + tokens, kv, dim), generator=gen).double() * 2 - 1
    q[..., :4] = k[..., :4] = LARGE
    k[..., 4:32] = 0
    around = torch.rand(tokens, heads, generator=gen).double() * 16 - 8
    lse = ((4 * LARGE ** 2 + around) * scale).float()
    x = torch.einsum("ihd,phd->ihp", q, k.repeat_interleave(heads // kv, 1))
    sees = torch.arange(START + tokens) <= START + torch.arange(tokens)[:, None, None]
    return q, k, lse, x, sees.expand(x.shape)


def _sums(w, kv):
    tokens, heads, keys = w.shape
    return w.view(tokens, kv, heads // kv, keys).sum((0, 2))


def _want(lse, x, sees, kv, scale):
    t = x * scale - lse.double()[..., None]
    w = torch.where(sees, torch.exp(t), 0)
    off = w * (2 * 2.0 ** -24 * t.abs() + 2 * 2.0 ** -22 + 2.0 ** -30)
    columns = x.shape[0] * x.shape[1] // kv
    return _sums(w, kv), _sums(off, kv) + (columns + 16) * 2.0 ** -24 * _sums(w, kv)


CASES = ((28, 4, 128, 1), (28, 4, 128, 2), (16, 4, 256, 3), (28, 4, 128, 20), (16, 4, 256, 70),
         (16, 2, 128, 90), (16, 2, 256, 90))


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("heads,kv,dim,tokens", CASES)
def test_the_bound_tells_roundings_apart(heads, kv, dim, tokens, scale):
    """The bound holds for the correction e = (s / s' - 1) L' - (L - L'), and not without it, with its
    sign wrong, or with either half of it alone."""
    _, _, lse, x, sees = _inputs(heads, kv, dim, tokens, scale)
    want, off = _want(lse, x, sees, kv, scale)
    assert torch.tensor(scale).double() == scale and x.max() < 2 ** 24
    log2e = 1 / math.log(2)
    s, l = scale * log2e, lse.double() * log2e
    s_near, l_near = float(torch.tensor(s).float()), l.float().double()
    rest, lo = s / s_near - 1, l - l_near
    assert 0.99 * 2.0 ** -24 < abs(rest) < 2.0 ** -24
    for e, right in ((rest * l_near - lo, True), (0 * lo, False), (lo - rest * l_near, False),
                     (-lo, False), (rest * l_near, False)):
        w = torch.where(sees, torch.exp2(s_near * x - l_near[..., None] + e[..., None]), 0)
        wrong = (_sums(w, kv) - want).abs() / off
        if right:
            assert wrong.max() < 0.5
        else:
            assert wrong.amax() > 2


def _cache(k, kv, dim, bits):
    keys = k.shape[0]
    width = -(-keys // 16)
    table = torch.randperm(width, generator=torch.Generator().manual_seed(width))
    rows = torch.zeros(width * 16, kv, dim, dtype=torch.float64)
    rows[:keys] = k
    rows = rows.view(width, 16, kv, dim).transpose(1, 2)
    place = table[None].int().cuda()
    if bits == 16:
        pages = torch.empty(width, kv, 16, dim, dtype=torch.bfloat16)
        pages[table] = rows.to(torch.bfloat16)
        assert torch.equal(pages[table].double(), rows)
        return paged.PagedCache(pages.cuda(), torch.zeros_like(pages).cuda()), place
    # 6 at a scale of 2^4, and 1, 0 or -1
    code = (rows.abs() == LARGE) * 7 + (rows.abs() == 1) * 2 + (rows < 0) * 8
    raw = torch.empty(width, kv, 16, dim // 2, dtype=torch.uint8)
    raw[table] = (code[..., ::2] | code[..., 1::2] << 4).to(torch.uint8)
    scales = torch.full((width, kv, 16, dim // 32), 127, dtype=torch.uint8)
    scales[..., 0] = 131
    return paged.PagedCache(raw.cuda(), torch.zeros_like(raw).cuda(), scales.cuda(),
                            scales.clone().cuda()), place


@pytest.mark.gpu
@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("heads,kv,dim,tokens", CASES)
def test_weights_of_large_scores(gpu, heads, kv, dim, tokens, scale, bits):
    q, k, lse, x, sees = _inputs(heads, kv, dim, tokens, scale)
    want, off = _want(lse, x, sees, kv, scale)
    cache, table = _cache(k, kv, dim, bits)
    weights = torch.zeros(1, kv, table.shape[1] * 16, device="cuda")
    start = torch.tensor([START], dtype=torch.int32, device="cuda")
    paged.accumulate_weights(weights, q[None].to(torch.bfloat16).cuda(), lse[None].cuda(), cache, table,
                             start, scale)
    got = weights[0].double().cpu()
    wrong = (got[:, :want.shape[1]] - want).abs() / off
    assert wrong.max() <= 1, wrong.max().item()
    assert (got[:, want.shape[1]:] == 0).all()
