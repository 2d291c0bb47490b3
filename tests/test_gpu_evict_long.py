"""Evictions of long rows, where ranks lie in LDS or are formed anew from weights and positions that
the same call rewrites: in place, behind an earlier eviction, rows of an odd stride."""

import pytest

import paged_reference as ref
from test_gpu_evict import _check_evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("moved,in_place", ((0, True), (1, True), (1, False)))
@pytest.mark.parametrize("keys,budget,bits", ((5000, 3100, 16), (32768, 9001, 4), (33001, 20000, 16),
                                              (50000, 777, 4)))
def test_evict_long_again(gpu, keys, budget, bits, moved, in_place):
    """`moved`: the first half of the shorter row's slots have positions, in no order."""
    s = ref.make(121, 2, 1, 2, 1, 128, 64, -(-keys // 64), (0, 0), bits=bits)
    lengths = (keys, keys - 333)
    seen = [n * 2 + 55 for n in lengths] if moved else None
    _check_evict(s, lengths, budget, budget // 7, 4, seen, moved * (keys - 333) // 2, 3, in_place)
