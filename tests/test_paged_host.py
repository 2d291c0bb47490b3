"""The paged cache on the host: what the functions and the C entry points refuse, before any
launch, and the 64-bit reference's 4-bit grid against its definition."""

import ctypes
import struct

import pytest
import torch

from exp3_amd import _lib, paged
import paged_reference as ref

FAKE, OFF = 1 << 20, (1 << 20) + 8
S4 = bytes((ctypes.c_int64 * 4)(4096, 512, 128, 1))
ODD = bytes((ctypes.c_int64 * 4)(4096, 512, 132, 1))


def _cache(pages=(FAKE, FAKE, 0, 0), table=FAKE, starts=FAKE, counts=0, stride=32, width=32, held=64,
           page_size=128, kv_heads=4, dim=128, batch=2, tokens=1, reserved=0):
    return struct.pack("7Pq8i", *pages, table, starts, counts, stride, width, held, page_size,
                       kv_heads, dim, batch, tokens, reserved)


def _append(cache=None, q=FAKE, k=FAKE, ks=S4, q_heads=28, cos=FAKE, sin=FAKE, rope=(4096, 128, 0),
            q_out=FAKE, k_out=None, **more):
    return _lib.load().spx_paged_append(cache or _cache(**more), q, S4, k, ks, FAKE, S4, q_heads, cos,
                                        sin, *rope, q_out, k_out, None)


def _gather(out=FAKE, **more):
    return _lib.load().spx_paged_gather(_cache(**more), out, FAKE, None)


def _attention(q=FAKE, qs=S4, q_heads=28, max_keys=0, workspace=FAKE, out=FAKE, **more):
    return _lib.load().spx_paged_attention(_cache(**more), q, qs, q_heads, max_keys, 0.1, workspace,
                                           out, None, None)


@pytest.mark.parametrize("call", (_append, _gather, _attention))
def test_shared_arguments(call):
    unsupported, invalid = _lib.SPX_EUNSUPPORTED, _lib.SPX_EINVAL
    for size in (8, 24, 100, 2048):
        assert call(page_size=size) == unsupported and b"page_size" in _lib.load().spx_last_error()
    assert call(dim=64) == unsupported
    assert call(batch=0) == call(tokens=0) == call(kv_heads=0) == call(held=0) == invalid
    assert call(table=0) == call(width=0) == call(starts=0) == invalid
    assert call(kv_heads=(1 << 16) + 4) == call(reserved=1) == invalid
    assert call(width=(1 << 23) + 1) == invalid                   # 2^30 + 128 positions
    for pages in ((0, FAKE, 0, 0), (FAKE, OFF, 0, 0), (FAKE, FAKE, FAKE, 0),
                  (FAKE, FAKE, FAKE, FAKE + 4)):
        assert call(pages=pages) == invalid
    assert call(table=FAKE + 2) == call(starts=FAKE + 1) == call(counts=FAKE + 2) == invalid


def test_append_arguments():
    unsupported, invalid = _lib.SPX_EUNSUPPORTED, _lib.SPX_EINVAL
    assert _lib.load().spx_paged_append(None, *[None] * 6, 0, None, None, 0, 0, 0, None, None,
                                        None) == invalid
    assert _append(k=None) == _append(k=OFF) == _append(ks=ODD) == invalid
    assert _append(q_out=None) == _append(k_out=OFF) == _append(q=OFF) == _append(q_heads=0) == invalid
    assert _append(sin=None) == _append(cos=OFF) == invalid
    assert _append(rope=(4095, 128, 0)) == invalid                # the table reaches 4096
    for rotary in (0, 8, 120, 144):
        assert _append(rope=(4096, rotary, 0)) == unsupported
    assert _append(tokens=(1 << 24) + 1) == _append(q_heads=1 << 20) == invalid


def test_gather_and_attention_arguments():
    invalid = _lib.SPX_EINVAL
    assert _gather(out=None) == _gather(out=OFF) == _gather(tokens=(1 << 24) + 1) == invalid
    assert _attention(q=None) == _attention(q=OFF) == _attention(qs=ODD) == invalid
    assert _attention(out=None) == _attention(max_keys=-1) == _attention(workspace=None) == invalid
    assert _attention(q_heads=27) == _attention(batch=1 << 16, tokens=1 << 10, q_heads=32) == invalid
    # units of 128 keys are counted in 32 bits: 2^23 of a table's reach for 256 streams
    assert _attention(width=1 << 23, batch=64) == invalid and b"bad shape" in _lib.load().spx_last_error()
    size = _lib.load().spx_paged_attention_workspace_bytes
    assert size(_cache(), 28, 0) > 0 and size(_cache(), 28, 100) == 0
    assert size(None, 28, 0) == size(_cache(), 27, 0) == size(_cache(), 28, -1) == -1
    assert size(_cache(batch=0), 28, 0) == size(_cache(dim=64), 28, 0) == -1


def test_wrappers_refuse():
    cache = paged.empty_pages(4, 16, 2, 128, "cpu")
    x = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    table, starts = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: paged.append_tokens(cache, table, starts, x, x),
                 lambda: _lib.host_module().append(*[cache.key_pages, cache.value_pages, None, None],
                                                   table, starts, None, x, x, *[None] * 3, 0, 0, 0),
                 lambda: _lib.host_module().gather(cache.key_pages, cache.value_pages, None, None,
                                                   table, starts, None, 1, 0),
                 lambda: _lib.host_module().attention(cache.key_pages, cache.value_pages, None, None,
                                                      table, starts, None, x, 0.1, 0, 0, 0),
                 lambda: paged.gather_tokens(cache, table, starts, 1),
                 lambda: paged.paged_attention(x, cache, table, starts, 0.1)):
        with pytest.raises(ValueError, match="ROCm GPU"):
            call()
    for bad in ((4, 8, 2, 128), (4, 24, 2, 128), (4, 2048, 2, 128), (4, 16, 2, 64)):
        with pytest.raises(ValueError, match="unsupported"):
            paged.empty_pages(*bad, "cpu")


def _describe(cache, table, starts, counts, batch=2, tokens=3):
    return _lib.host_module().describe(cache.key_pages, cache.value_pages, cache.key_scales,
                                       cache.value_scales, table, starts, counts, batch, tokens)


def test_checks_of_the_host_module():
    """Its checks of cache and page table, which look at no device, on the CPU."""
    good = paged.empty_pages(4, 16, 2, 128, "cpu", four_bit=True)
    half = paged.empty_pages(4, 16, 2, 256, "cpu")
    table, starts = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    assert _describe(good, table, starts, starts) == (4, 16, 2, 128, 4)
    assert _describe(half, table, starts, None) == (4, 16, 2, 256, 4)
    assert (good.page_size, good.kv_heads, good.head_dim, good.four_bit) == (16, 2, 128, True)
    assert half.head_dim == 256 and not half.four_bit
    bad = (paged.PagedCache(good.key_pages, good.value_pages, good.key_scales),
           paged.PagedCache(half.key_pages, half.value_pages, None, good.value_scales),
           paged.PagedCache(good.key_pages, good.value_pages),
           paged.PagedCache(half.key_pages, half.value_pages[:3]),
           paged.PagedCache(half.key_pages.transpose(1, 2), half.value_pages.transpose(1, 2)),
           paged.PagedCache(half.key_pages.half(), half.value_pages.half()),
           paged.PagedCache(half.key_pages[0], half.value_pages[0]),
           paged.PagedCache(half.key_pages, None), paged.PagedCache(None, half.value_pages),
           paged.PagedCache(good.key_pages, good.value_pages, good.key_scales[..., :2],
                            good.value_scales[..., :2]),
           paged.PagedCache(half.key_pages, half.value_pages.to("meta")))
    for cache in bad:
        with pytest.raises(ValueError):
            _describe(cache, table, starts, None)
    assert _describe(good, torch.zeros(2, 9, dtype=torch.int32)[:, 2:6], starts, None)[-1] == 4
    for wrong in ((table.long(), starts, None), (table, starts.long(), None), (table[:1], starts, None),
                  (table, starts[:1], None), (table, starts, starts.long()), (table[0], starts, None),
                  (table.repeat(1, 2)[:, ::2], starts, None), (table, starts[:, None], None),
                  (table, torch.zeros(4, dtype=torch.int32)[::2], None), (table, None, None),
                  (table, starts, [0, 0])):
        with pytest.raises(ValueError):
            _describe(good, *wrong)
    with pytest.raises(TypeError):
        _lib.host_module().describe(1, 2)


def test_rope_table_far_positions():
    cos, sin = paged.rope_table(131072, 128)
    angle = torch.tensor(131071.0, dtype=torch.float64) * \
        1.0e6 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    # one rounding to fp32 of a value that fp64 has to 131072 x 2^-52
    assert (cos[-1].double() - angle.cos()).abs().max() <= 2.0 ** -25 + 2.0 ** -34
    assert (sin[-1].double() - angle.sin()).abs().max() <= 2.0 ** -25 + 2.0 ** -34
    assert cos.shape == sin.shape == (131072, 64) and cos.dtype == torch.float32


def test_reference_grid():
    """Each value against all representable ones: none is nearer, ties have an even code."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(40, 32, generator=gen, dtype=torch.float64)
    x[0, :17] = torch.tensor([0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 6.9, -.25, -.75, -2.5, -5,
                              0.2500001, 2.4999, -0.0])
    x[0, 17:] = 0.1
    got = ref.four_bit(x)
    assert got[0, :17].tolist() == [0, 0, 1, 1, 2, 2, 4, 4, 6, 6, 0, -1, -2, -4, 0.5, 2, 0]
    top = x.abs().amax(-1)
    step = 2.0 ** torch.ceil(torch.log2(top / 7))
    step = torch.where(top / step >= 7, step * 2, step)
    near = ((x.abs() / step[:, None])[..., None] - ref.GRID).abs().amin(-1)
    assert torch.equal((x - got).abs() / step[:, None], near)
    assert torch.equal(ref.four_bit(torch.zeros(1, 32)), torch.zeros(1, 32, dtype=torch.float64))
    wild = torch.zeros(2, 64)
    wild[0, 3], wild[1, 40] = float("inf"), float("nan")
    out = ref.four_bit(wild)
    assert torch.isnan(out[0, :32]).all() and torch.isnan(out[1, 32:]).all()
    assert (out[0, 32:] == 0).all() and (out[1, :32] == 0).all()
    assert ref.four_bit(torch.full((1, 32), 3.3e38, dtype=torch.float64)).max() == 6 * 2.0 ** 125


@pytest.mark.parametrize("which", (0, 1))
def test_pages_that_require_a_gradient(which):
    """Refused while gradients are recorded, as q, k and v: no output would carry one."""
    cache = paged.empty_pages(4, 16, 2, 128, "cpu")
    table, starts = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    page = (cache.key_pages, cache.value_pages)[which].requires_grad_()
    with pytest.raises(ValueError, match="requires a gradient"):
        _describe(cache, table, starts, None)
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            _describe(cache, table, starts, None)
    page.requires_grad_(False)
    _describe(cache, table, starts, None)


@pytest.mark.parametrize("which", (0, 1))
def test_pages_with_a_forward_tangent(which):
    """Refused: the tangent would be dropped."""
    cache = paged.empty_pages(4, 16, 2, 128, "cpu")
    table, starts = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    pages = [cache.key_pages, cache.value_pages]
    with torch.autograd.forward_ad.dual_level():
        _describe(cache, table, starts, None)
        pages[which] = torch.autograd.forward_ad.make_dual(pages[which], torch.ones_like(pages[which]))
        dual = paged.PagedCache(*pages)
        with pytest.raises(ValueError, match="tangent"):
            _describe(dual, table, starts, None)
        pages[which] = torch.autograd.forward_ad.unpack_dual(pages[which]).primal
        _describe(paged.PagedCache(*pages), table, starts, None)


def test_refused_while_a_graph_is_traced():
    """torch records the outputs' allocation and not the kernel: what was traced would return
    uninitialised memory."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode

    cache = paged.empty_pages(4, 16, 2, 128, "cpu")
    table, starts = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)

    def step(x):
        _describe(cache, table, x, None)
        return x + 1

    step(starts)
    with FlopCounterMode(display=False):          # a mode that only looks on
        step(starts)
    for trace in (lambda: torch.jit.trace(step, (starts,)), lambda: make_fx(step)(starts),
                  lambda: make_fx(step, tracing_mode="fake")(starts)):
        with pytest.raises(ValueError, match="traced"):
            trace()
    with FakeTensorMode(), pytest.raises(ValueError, match="traced"):
        _describe(cache, table, starts, None)
    step(starts)


class _Wrapped(torch.Tensor):
    """A subclass that computes by itself."""

    @classmethod
    def __torch_dispatch__(cls, function, types, args=(), kwargs=None):
        raise AssertionError("not called")


def test_tensors_that_are_not_their_storage():
    """Lazily negated or zero tensors and subclasses: the kernels would read something else."""
    for four in (False, True):
        cache = paged.empty_pages(4, 16, 2, 128, "cpu", four_bit=four)
        table, starts = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
        good = [cache.key_pages, cache.value_pages, cache.key_scales, cache.value_scales, table, starts,
                starts.clone()]

        def describe(*args):
            return _describe(paged.PagedCache(*args[:4]), *args[4:])

        describe(*good)
        for i, x in enumerate(good):
            if x is None:
                continue
            for other in (torch._neg_view(x), torch._efficientzerotensor(x.shape, dtype=x.dtype),
                          torch.Tensor._make_subclass(_Wrapped, x)):
                with pytest.raises(ValueError, match="plain"):
                    describe(*good[:i], other, *good[i + 1:])
    param = torch.nn.Parameter(cache.key_scales, requires_grad=False)     # plain for all that
    describe(*good[:2], param, *good[3:])

    def functional(x):
        with pytest.raises(ValueError, match="plain"):
            describe(*good[:6], x)
        return x

    torch.func.functionalize(functional)(starts)


def test_more_streams_than_one_launch_of_workgroups():
    """2^32 threads and more do not fit a launch of one workgroup of 512 per stream: such calls share
    their units, which takes a workspace. More heads than a join's launch has threads for: refused."""
    size = _lib.load().spx_paged_attention_workspace_bytes
    few = dict(width=4, page_size=128, kv_heads=8)               # 512 positions
    assert size(_cache(batch=(1 << 20) - 1, **few), 8, 0) == 0
    for batch in (1 << 20, 1 << 21):
        assert size(_cache(batch=batch, **few), 8, 0) > batch * 8 * 8
        assert size(_cache(batch=batch, **few), 8, 300) > batch * 8 * 8
    assert size(_cache(batch=1, width=32, kv_heads=1 << 16), 1 << 20, 0) > 0
    assert size(_cache(batch=1, width=32, kv_heads=1 << 16), 1 << 21, 0) == -1
    assert _attention(batch=1, kv_heads=1 << 16, q_heads=1 << 21) == _lib.SPX_EINVAL


def test_rope_table_sizes():
    """rotary_dim is a number of dims that pair: an odd one gave a table of other angles."""
    for size in (127, 1, 0, -2):
        with pytest.raises(ValueError, match="rotary_dim"):
            paged.rope_table(16, size)


def test_wrappers_refuse_what_is_no_tensor():
    cache = paged.empty_pages(4, 16, 2, 128, "cpu")
    for x in (None, [1], 2.0):
        for call in (lambda: paged.append_tokens(cache, None, None, x, x),
                     lambda: paged.gather_tokens(cache, x, None, 1),
                     lambda: paged.paged_attention(x, cache, None, None, 0.1)):
            with pytest.raises(ValueError, match="tensor"):
                call()


@pytest.mark.parametrize("call", (_append, _gather))
def test_batches_near_the_end_of_32_bits(call):
    """Refused before the launch, whose size a batch above 2^31 - 65535 overflowed."""
    for batch in (2**31 - 1, (1 << 30) + 1):
        assert call(batch=batch) == _lib.SPX_EINVAL and b"2^30" in _lib.load().spx_last_error()
