"""Drafted trees and gathered weights of more sequences than a wave looks at at once (64)."""

import pytest
import torch

import paged_reference as ref
from test_gpu_evict import _check_weights
from test_gpu_trees import _check, _tree

pytestmark = pytest.mark.gpu


def _starts(batch, free, most):
    """Ragged; free slots first, last and in between."""
    starts = [(37 * b) % most for b in range(batch)]
    for b in list(range(free)) + [batch // 2, batch - 1]:
        starts[b] = -1
    return tuple(starts)


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("batch,free,layout,tokens", ((65, 64 - 1, (8, 2, 128), 5), (130, 0, (8, 2, 128), 5),
                                                      (130, 70, (28, 4, 128), 3), (200, 3, (4, 2, 256), 9),
                                                      (129, 127, (8, 8, 128), 20)))
def test_tree_of_many_sequences(gpu, batch, free, layout, tokens, bits):
    starts = list(_starts(batch, free, 300))
    if free > batch // 2:
        starts[-1] = 250                                           # the only one, or one of a few
    s = ref.make(131, batch, tokens, *layout, 16, 20, tuple(starts), bits=bits)
    _check(s, _tree(131, batch, tokens), 0.1)


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("batch,free,layout,tokens", ((130, 0, (8, 2, 128), 1), (200, 66, (8, 2, 128), 4),
                                                      (130, 2, (4, 1, 256), 2), (100, 65, (8, 2, 128), 20),
                                                      (70, 1, (8, 1, 128), 66)))
def test_weights_of_many_sequences(gpu, batch, free, layout, tokens, bits):
    """Few columns, whole blocks of keys, and (528 columns) blocks that workgroups share."""
    s = ref.make(132, batch, tokens, *layout, 16, 18, _starts(batch, free, 220), bits=bits)
    first, _ = _check_weights(s, 0.1)
    again, _ = _check_weights(s, 0.1)
    assert torch.equal(first, again)
