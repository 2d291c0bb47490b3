"""Paged attention of more streams than one launch has workgroups of 512 threads."""

import pytest
import torch

from exp3_amd import paged
import paged_reference as ref

pytestmark = pytest.mark.gpu


def test_attention_of_a_million_sequences(gpu):
    """2^20 sequences of 8 KV heads over a reach of 64 tokens: 2^23 streams, 2^32 threads if each had
    a workgroup of its own. Every fourth sequence is the same."""
    s = ref.make(30, 4, 1, 8, 8, 128, 16, 4, (40, -1, 0, 63), spare=0)
    want, want_lse, off, lse_off = (x.cuda() for x in ref.attention(s, 0.1))
    cache, table, starts, _ = ref.on_gpu(s)
    times = 1 << 18
    q, table, starts = (x.repeat(times, *([1] * (x.dim() - 1))) for x in (s.q.cuda(), table, starts))
    out, lse = paged.paged_attention(q, cache, table, starts, 0.1, return_lse=True)
    first, first_lse = out[:4].clone(), lse[:4].clone()
    assert ((first.double() - want).abs() <= 2.0 ** -8 * want.abs() + off).all()
    assert ((first_lse == want_lse) | ((first_lse - want_lse).abs() <= lse_off)).all()
    assert (out.view(times, *first.shape) == first).all()
    assert (lse.view(times, *first_lse.shape) == first_lse).all()
