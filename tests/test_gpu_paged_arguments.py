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


def test_forward_tangents(gpu):
    """Refused wherever they come in: the outputs would carry none."""
    cache, table, starts, x, rope = _call()

    def dual(y):
        return torch.autograd.forward_ad.make_dual(y, torch.ones_like(y))

    with torch.autograd.forward_ad.dual_level():
        paged.append_tokens(cache, table, starts, x, x, x, rope)
        pages = paged.PagedCache(dual(cache.key_pages), cache.value_pages)
        for call in (lambda: paged.append_tokens(cache, table, starts, dual(x), x),
                     lambda: paged.append_tokens(cache, table, starts, x, dual(x)),
                     lambda: paged.append_tokens(cache, table, starts, x, x, dual(x)),
                     lambda: paged.append_tokens(cache, table, starts, x, x, x, (rope[0], dual(rope[1]))),
                     lambda: paged.append_tokens(pages, table, starts, x, x),
                     lambda: paged.gather_tokens(pages, table, starts, 1),
                     lambda: paged.paged_attention(x, pages, table, starts, 0.1),
                     lambda: paged.paged_attention(dual(x), cache, table, starts, 0.1)):
            with pytest.raises(ValueError, match="tangent"):
                call()
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(lambda y: paged.paged_attention(y, cache, table, starts, 0.1), (x,), (x,))
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.grad(lambda y: paged.paged_attention(y, cache, table, starts, 0.1).sum())(x)
    with pytest.raises((ValueError, RuntimeError)):
        torch.vmap(lambda y: paged.paged_attention(y, cache, table, starts, 0.1))(x[None].expand(2, -1, -1, -1, -1))


def test_refused_while_a_graph_is_traced(gpu):
    """torch records the outputs' allocation and not the kernel: what was traced would return
    uninitialised memory. A compiled function takes the calls as they are."""
    from torch.fx.experimental.proxy_tensor import make_fx

    cache, table, starts, x, rope = _call()
    for step in (lambda y: paged.append_tokens(cache, table, starts, y, y, y, rope)[0],
                 lambda y: paged.gather_tokens(cache, table, starts, 1)[0] + y,
                 lambda y: paged.paged_attention(y, cache, table, starts, 0.1)):
        want = step(x)
        for trace in (lambda: torch.jit.trace(step, (x,)), lambda: make_fx(step)(x)):
            with pytest.raises(ValueError, match="traced"):
                trace()
        assert torch.equal(torch.compile(step, backend="eager")(x), want)


def test_tensors_that_are_not_their_storage(gpu):
    """Lazily negated rope tables are refused, queries, keys and values are read with the sign; lazily
    zero ones are refused."""
    cache, table, starts, x, rope = _call()
    want = [*paged.append_tokens(cache, table, starts, x, x, x, rope, return_keys=True),
            cache.key_pages.clone(), cache.value_pages.clone()]
    minus = torch._neg_view(-x)
    got = [*paged.append_tokens(cache, table, starts, minus, minus, minus, rope, return_keys=True),
           cache.key_pages, cache.value_pages]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(paged.paged_attention(minus, cache, table, starts, 0.1),
                       paged.paged_attention(x, cache, table, starts, 0.1))
    for i in range(2):
        for other in (torch._neg_view(rope[i]),
                      torch._efficientzerotensor(rope[i].shape, dtype=torch.float32, device="cuda")):
            with pytest.raises(ValueError, match="plain"):
                paged.append_tokens(cache, table, starts, x, x, x, (other, rope[1]) if i == 0 else
                                    (rope[0], other))
    zero = torch._efficientzerotensor(x.shape, dtype=x.dtype, device="cuda")
    for call in (lambda: paged.append_tokens(cache, table, starts, zero, x),
                 lambda: paged.append_tokens(cache, table, starts, x, zero),
                 lambda: paged.append_tokens(cache, table, starts, x, x, zero),
                 lambda: paged.paged_attention(zero, cache, table, starts, 0.1)):
        with pytest.raises(ValueError, match="plain"):
            call()


@pytest.mark.parametrize("four", (False, True))
def test_append_counts_as_a_write(gpu, four):
    """The versions by which autograd finds that a saved tensor was written over: those of the pages
    and scales that an append writes, and no others."""
    _, table, starts, x, rope = _call()
    cache = paged.empty_pages(8, 16, 2, 128, "cuda", four_bit=four)
    tensors = [t for t in vars(cache).values() if t is not None] + [table, starts, x, *rope]
    before = [t._version for t in tensors]
    paged.gather_tokens(cache, table, starts, 1)
    paged.paged_attention(x, cache, table, starts, 0.1)
    paged.append_tokens(cache, table, starts, x[:, :0], x[:, :0])
    assert [t._version for t in tensors] == before
    paged.append_tokens(cache, table, starts, x, x, x, rope)
    written = 4 if four else 2
    assert all(t._version > v for t, v in zip(tensors[:written], before))
    assert [t._version for t in tensors[written:]] == before[written:]
    if not four:
        leaf = torch.ones((), device="cuda", dtype=torch.bfloat16, requires_grad=True)
        product = (cache.key_pages * leaf).sum()
        paged.append_tokens(cache, table, starts, x, x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()
    with torch.inference_mode():               # tensors without a version
        inner = paged.empty_pages(8, 16, 2, 128, "cuda", four_bit=four)
        paged.append_tokens(inner, table, starts, x, x)
    paged.append_tokens(inner, table, starts, x, x)
