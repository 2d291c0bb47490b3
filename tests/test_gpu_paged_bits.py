"""Probabilities and their sums in paged attention hold 32 bits: keys whose scores are exact, so that
nothing but the exponential, the sums and the logarithm rounds, in every form of the kernel."""

import math

import pytest
import torch

from exp3_amd import paged
import paged_reference as ref

pytestmark = pytest.mark.gpu

KEY = -0.75          # of the keys with a probability below 1, in dim 0
DIGITS = 9


def _parts(p):
    """p in two bf16 parts, and what they leave of it in fp32."""
    p = p.float()
    high = p.bfloat16().float()
    low = (p - high).bfloat16().float()
    return (high + low).double(), (p - high - low).double()


def _queries(count):
    """Values of dim 0 in [1/2, 1) whose probabilities exp(KEY q) two bf16 parts hold worst."""
    q = (0.5 + torch.arange(128) / 256).double()
    left = _parts(torch.exp(KEY * q))[1].abs()
    worst = q[left.argsort(descending=True)[:count]]
    assert _parts(torch.exp(KEY * worst))[1].abs().min() > 2.0 ** -18.7
    return worst


def _call(layout, bits, reach, below):
    """One sequence whose first keys score 0 or KEY q (`below`: which), one token behind them; values 0;
    a table that reaches `reach` positions."""
    q_heads, kv_heads, dim = layout
    keys = len(below)
    s = ref.make(1, 1, 1, q_heads, kv_heads, dim, 16, 1, (keys - 1,), bits=bits, spare=0)
    s.table = s.table.repeat(1, reach // 16)
    group = q_heads // kv_heads
    s.q.zero_()
    s.q[0, 0, :, 0] = _queries(group).repeat(kv_heads).to(torch.bfloat16)
    rows = torch.zeros(1, kv_heads, 16, dim, dtype=torch.float64)
    rows[0, :, :keys, 0] = KEY * torch.tensor(below).double()
    _fill(s, 0, rows)
    _fill(s, 1, torch.zeros_like(rows))
    return s


def _fill(s, which, rows, step=None):
    """Rows of the cache; 4 bits: multiples of `step` by grid values (KEY is 3 x 2^-2)."""
    if s.bits == 16:
        s.held[which] = rows.to(torch.bfloat16)
        return
    step = torch.full((*rows.shape[:3], 1), 0.25, dtype=torch.float64) if step is None else step
    near = (rows.abs() / step)[..., None] - ref.GRID
    assert (near == 0).any(-1).all()
    code = (near == 0).to(torch.uint8).argmax(-1).to(torch.uint8) | (rows < 0).to(torch.uint8) << 3
    s.raw[which] = code[..., ::2] | code[..., 1::2] << 4
    scale = (127 + torch.log2(step)).to(torch.uint8)
    s.scales[which] = scale.expand(*rows.shape[:3], rows.shape[3] // 32).contiguous()
    s.held[which] = ref.values(s.raw[which], s.scales[which])
    assert torch.equal(s.held[which], rows)


# one workgroup per stream; shared units; many of them (two columns' sets in one tile at 8 heads and less)
FORMS = [(layout, bits, reach) for layout in ((28, 4, 128), (8, 8, 128), (16, 4, 256))
         for bits in (16, 4) for reach in (64, 4096, 262144)]


@pytest.mark.parametrize("layout,bits,reach", FORMS)
def test_lse(gpu, layout, bits, reach):
    """One key of score 0, fifteen of KEY q. In units of 2^-24: the exponent (below 1.04, the scale's
    rounding and its own) 1.5 and the exponential's ulp 2 of each probability, at most 20 additions of
    an ulp each 40, the logarithm (below 4, an ulp) 2.8, its product with ln 2 2. Sums of two bf16 parts
    would be off by 67 or more."""
    s = _call(layout, bits, reach, [0] + [1] * 15)
    cache, table, starts, _ = ref.on_gpu(s)
    _, lse = paged.paged_attention(s.q.cuda(), cache, table, starts, 1.0, return_lse=True)
    want = ref.attention(s, 1.0)[1]
    two = torch.log1p(15 * _parts(torch.exp(KEY * s.q[0, 0, :, 0].double()))[0])
    assert (two - want[0, 0]).abs().max() > 67 * 2.0 ** -24     # such a sum fails this test
    off = (lse.double().cpu() - want).abs().max().item()
    assert off <= 49 * 2.0 ** -24, off * 2.0 ** 24


@pytest.mark.parametrize("layout,bits,reach", FORMS)
def test_output(gpu, layout, bits, reach):
    """Keys of score 0 whose values add up to minus the two bf16 parts of one head's probability, in
    dims of its own, and one key of that probability with the value 1: what is left is the third
    part over the sum of the probabilities, 9 and one below 1. The sum of the products is off by the
    probability's error (below 1: 1.5 for its exponent, 1 ulp) and at most 10 additions of magnitudes
    of 2 and less, an ulp of 2 each: 2.5 + 20 units of 2^-24, over 9."""
    s = _call(layout, bits, reach, [0] * DIGITS + [1])
    group, groups = layout[0] // layout[1], layout[2] // 32
    heads = min(group, groups)
    rows = torch.zeros(1, layout[1], 16, layout[2], dtype=torch.float64)
    step = torch.full((1, layout[1], 16, 1), 1.0, dtype=torch.float64)
    held = _parts(torch.exp(KEY * s.q[0, 0, :heads, 0].double()))[0]
    for h in range(heads):
        rest = int(held[h] * 4 ** DIGITS)
        assert rest == held[h] * 4 ** DIGITS
        for j in range(DIGITS):                       # digits of base 4
            digit, rest = divmod(rest, 4 ** (DIGITS - 1 - j))
            rows[0, :, j, 32 * h:32 * h + 32] = -digit * 4.0 ** -(j + 1)
            step[0, :, j] = 4.0 ** -(j + 1)
        rows[0, :, DIGITS, 32 * h:32 * h + 32] = 1
    _fill(s, 1, rows, step)
    cache, table, starts, _ = ref.on_gpu(s)
    out = paged.paged_attention(s.q.cuda(), cache, table, starts, 1.0).double().cpu()
    want = ref.attention(s, 1.0)[0]
    for h in range(layout[0]):
        if h % group >= heads:
            continue
        dims = slice(32 * (h % group), 32 * (h % group) + 32)
        got, right = out[0, 0, h, dims], want[0, 0, h, dims]
        assert right.abs().min() > 22.5 / 9 * 2.0 ** -24 + 2.0 ** -22.6     # 0 fails this test
        off = ((got - right).abs() - 2.0 ** -8 * right.abs()).max().item()
        assert off <= 22.5 / 9 * 2.0 ** -24, (h, off * 2.0 ** 24)
        assert math.copysign(1, got[0]) == math.copysign(1, right[0])
