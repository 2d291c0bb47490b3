"""What the paged cache's functions take and refuse of tensors on the GPU beyond their shapes and
types."""

import pytest
import torch

from exp3_amd import paged

pytestmark = pytest.mark.gpu


def _call(rotary=128):
    """A cache of zeros, its page table, starts, one token and a rope table."""
    cache = paged.empty_pages(8, 16, 2, 128, "cuda")
    cache.key_pages.zero_()
    cache.value_pages.zero_()
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    starts = torch.full((1,), 5, dtype=torch.int32, device="cuda")
    x = torch.randn(1, 1, 2, 128, device="cuda").to(torch.bfloat16)
    return cache, table, starts, x, paged.rope_table(64, rotary, device="cuda")


@pytest.mark.parametrize("which", ("key_pages", "value_pages"))
def test_pages_that_require_a_gradient(gpu, which):
    cache, table, starts, x, _ = _call()
    getattr(cache, which).requires_grad_()
    for call in (lambda: paged.append_tokens(cache, table, starts, x, x),
                 lambda: paged.gather_tokens(cache, table, starts, 1),
                 lambda: paged.paged_attention(x, cache, table, starts, 0.1)):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("which", (0, 1))
def test_rope_tables_that_require_a_gradient(gpu, which):
    cache, table, starts, x, rope = _call()
    rope[which].requires_grad_()
    with pytest.raises(ValueError, match="requires a gradient"):
        paged.append_tokens(cache, table, starts, x, x, x, rope)
    with torch.no_grad():
        paged.append_tokens(cache, table, starts, x, x, x, rope)
