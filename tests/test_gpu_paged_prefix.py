"""A prompt that continues a cached prefix: append_tokens, then paged_attention of the whole chunk."""

import pytest
import torch

from exp3_amd import attention, paged
import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", (16, 4))
@pytest.mark.parametrize("prefix,chunk", ((300, 70), (1300, 129), (5, 2)))
def test_chunk_behind_a_prefix(gpu, prefix, chunk, bits):
    """Two sequences, the second with one prefix token and half the chunk: each new token sees the
    prefix and the chunk up to itself, as a prefill of the whole prompt does."""
    heads, dim, scale = (28, 4, 4), 128, 128 ** -0.5
    total = prefix + chunk
    gen = torch.Generator("cuda").manual_seed(prefix)
    fused = torch.randn(2, total, 36, dim, generator=gen, device="cuda").to(torch.bfloat16)
    width = -(-total // 16)
    cache = paged.empty_pages(2 * width, 16, 4, dim, "cuda", four_bit=bits == 4)
    table = torch.randperm(2 * width, generator=gen, device="cuda").view(2, width).int()
    rope = paged.rope_table(width * 16, dim, device="cuda")
    held, new = ([prefix, 1], [chunk, chunk // 2])
    starts, counts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (held, new))
    q, k, v = fused[:, :prefix].split(heads, 2)
    paged.append_tokens(cache, table, torch.zeros_like(starts), k, v, q, rope, starts)
    # the second sequence's chunk begins at its position 1
    rest = torch.stack((fused[0, prefix:], fused[1, 1:1 + chunk]))
    q, k, v = rest.split(heads, 2)
    q, _ = paged.append_tokens(cache, table, starts, k, v, q, rope, counts)
    out = paged.paged_attention(q, cache, table, starts, scale, counts)

    s = ref.make(0, 2, chunk, 28, 4, dim, 16, width, held, new, spare=0)
    s.q, s.table = q.cpu(), table.cpu()
    s.held = ref.contents(cache)
    want, _, off, _ = ref.attention(s, scale)
    assert ((out.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + off).all()
    assert not out[1, chunk // 2:].any()
    if bits == 16:
        # the backend's prefill of the whole first prompt rounds its probabilities to bf16 (an output
        # by 2^-8 of the largest value), both round their output
        q, k = paged.append_tokens(cache, table[:1], torch.zeros_like(starts[:1]), fused[:1, :, 28:32],
                                   fused[:1, :, 32:], fused[:1, :, :28], rope, return_keys=True)

        class Layer:
            layer_idx = 0

        whole, _ = attention.AttentionBackend(register=False, dense_impl="hip").forward(
            Layer(), *(x.transpose(1, 2) for x in (q, k, fused[:1, :, 32:])), None, scale)
        torch.testing.assert_close(out[0].float(), whole[0, prefix:].float(), rtol=2.0 ** -7,
                                   atol=2.0 ** -8 * fused.abs().max().item())
