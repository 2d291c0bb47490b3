"""Where an eviction's outputs may stand: in place, or in memory that no argument shares."""

import pytest
import torch

from exp3_amd import paged
import paged_reference as ref

pytestmark = pytest.mark.gpu


def _call():
    s = ref.make(101, 2, 1, 4, 2, 128, 16, 8, (0, 0))
    cache, table, _, _ = ref.on_gpu(s)
    gen = torch.Generator().manual_seed(101)
    shape = (2, 2, 128)
    room = torch.rand(4 * 512, generator=gen).cuda()             # four ledgers
    places = torch.full((4 * 512,), -1, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([120, 77], dtype=torch.int32, device="cuda")
    return cache, table, lengths, lambda x, at: x[at:at + 512].view(shape), room, places


def test_outputs_that_share_memory_are_refused(gpu):
    cache, table, lengths, view, room, places = _call()
    weights, positions = view(room, 512), view(places, 512)
    before = cache.key_pages.clone(), room.clone(), places.clone()
    for out in ((view(room, 513), view(places, 512)), (view(room, 1), view(places, 512)),
                (view(room, 512), view(places, 511)), (view(room, 512), view(places, 1023)),
                (view(places.view(torch.float32), 512), view(places, 0)),
                (view(room, 1024), view(room.view(torch.int32), 512)),
                (view(room, 1024), view(room.view(torch.int32), 1400))):
        with pytest.raises(ValueError, match="overlap"):
            paged.evict_tokens(cache, table, lengths, weights, 40, positions, out=out)
    long = torch.full((514,), 90, dtype=torch.int32, device="cuda")
    for name, more in (("lengths", {}), ("seen", dict(seen=long[512:]))):
        held = long[512:] if name == "lengths" else lengths
        with pytest.raises(ValueError, match="overlap"):
            paged.evict_tokens(cache, table, held, weights, 40, out=(weights, long[2:].view(2, 2, 128)),
                               **more)
    torch.cuda.synchronize()
    for x, y in zip((cache.key_pages, room, places), before):
        assert torch.equal(x, y)


def test_outputs_side_by_side(gpu):
    """In place, next to the arguments, and one of each kind: the same results."""
    got = []
    for at in ((512, 512), (0, 1024), (1024, 0), (512, 0), (0, 512)):
        cache, table, lengths, view, room, places = _call()
        out = view(room, at[0]), view(places, at[1])
        left, w, p = paged.evict_tokens(cache, table, lengths, view(room, 512), 40, view(places, 512),
                                        recent=5, sinks=2, out=out)
        assert w.data_ptr() == out[0].data_ptr() and p.data_ptr() == out[1].data_ptr()
        got.append([left, w.clone(), p.clone(), cache.key_pages, cache.value_pages])
    for other in got[1:]:
        assert all(torch.equal(x, y) for x, y in zip(got[0], other))


def test_a_cache_without_heads_is_refused(gpu):
    """No kernel would run, and nothing write the lengths that come back."""
    cache, table, lengths, *_ = _call()
    none = paged.PagedCache(cache.key_pages[:, :0], cache.value_pages[:, :0])
    with pytest.raises(ValueError, match="kv_heads"):
        paged.evict_tokens(none, table, lengths, torch.zeros(2, 0, 128, device="cuda"), 40)
