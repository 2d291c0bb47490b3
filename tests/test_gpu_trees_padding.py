"""Queries of rows that are no tokens, whatever they hold, change nothing in the rows that are."""

import math

import pytest
import torch

from exp3_amd import paged
import paged_reference as ref
import trees_reference as trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("tokens,layout", ((5, (8, 2, 128)), (20, (28, 4, 128)), (70, (28, 4, 128)),
                                           (9, (16, 4, 256)), (40, (16, 4, 256))))
@pytest.mark.parametrize("value", (math.nan, math.inf, -3.0e38))
def test_tree_queries_of_padding(gpu, tokens, layout, bits, value):
    """Behind the counts, past the table's end and in a free slot; bit for bit what zeros there give:
    the fp32 products of values that are not finite round otherwise."""
    reach = 16 * 60
    starts = (700, 333, reach - tokens // 2, -1, 0)
    counts = (max(tokens // 3, 1), tokens - 1, tokens, tokens, 0)
    s = ref.make(91, 5, tokens, *layout, 16, 60, starts, counts, bits=bits, sharp=2.0)
    cache, table, starts, counts = ref.on_gpu(s)
    masks = trees.words(trees.lineage(trees.random_parents(91, 5, tokens))[0]).cuda()
    got = []
    for filler in (0.0, value):
        q = s.q.clone()
        for b in range(5):
            q[b, trees.live_tokens(s, b):] = filler
        got.append(paged.tree_attention(q.cuda(), cache, table, starts, masks, 0.1, counts,
                                        return_lse=True))
    for x, y in zip(*got):
        assert torch.equal(x, y)
    assert torch.isfinite(got[0][0]).all()
