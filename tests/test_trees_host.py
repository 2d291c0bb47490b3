"""Drafted trees and evictions on the host: what the functions and the C entry points refuse, before
any launch."""

import ctypes

import pytest
import torch

from exp3_amd import _lib, paged
from test_paged_host import FAKE, ODD, OFF, S4, _cache

INVALID, UNSUPPORTED = _lib.SPX_EINVAL, _lib.SPX_EUNSUPPORTED


def _append_at(q=FAKE, k=FAKE, cos=FAKE, rope=(100, 128, 0), positions=FAKE, **more):
    return _lib.load().spx_paged_append_at(_cache(**more), q, S4, k, S4, FAKE, S4, 28, cos, cos, *rope,
                                           positions, FAKE, None, None)


def _tree(q=FAKE, qs=S4, q_heads=28, masks=FAKE, max_keys=0, workspace=FAKE, out=FAKE, **more):
    return _lib.load().spx_paged_tree_attention(_cache(**more), q, qs, q_heads, masks, max_keys, 0.1,
                                                workspace, out, None, None)


def _keep(caches=None, count=1, parents=FAKE, drafts=FAKE, targets=FAKE, path_in=None, accepted=FAKE,
          path_out=FAKE, following=FAKE, **more):
    return _lib.load().spx_paged_keep_path(caches or _cache(**more), count, parents, drafts, targets,
                                           path_in, accepted, path_out, following, None)


def _weights(q=FAKE, qs=S4, q_heads=28, lse=FAKE, workspace=FAKE, weights=FAKE, row=4096, **more):
    return _lib.load().spx_paged_accumulate_weights(_cache(**more), q, qs, q_heads, lse, 0.1, workspace,
                                                    weights, row, None)


def _evict(weights=FAKE, positions=None, row=4096, seen=None, budget=100, recent=4, sinks=2,
           workspace=FAKE, out=FAKE, positions_out=FAKE, lengths_out=FAKE, **more):
    return _lib.load().spx_paged_evict(_cache(**more), weights, positions, row, seen, budget, recent,
                                       sinks, workspace, out, positions_out, lengths_out, None)


@pytest.mark.parametrize("call", (_append_at, _tree, _keep, _weights, _evict))
def test_shared_arguments(call):
    for size in (8, 24, 100, 2048):
        assert call(page_size=size) == UNSUPPORTED and b"page_size" in _lib.load().spx_last_error()
    assert call(dim=64) == UNSUPPORTED
    assert call(batch=0) == call(tokens=0) == call(kv_heads=0) == call(held=0) == INVALID
    assert call(table=0) == call(width=0) == call(starts=0) == INVALID
    assert call(kv_heads=(1 << 16) + 4) == call(reserved=1) == INVALID
    for pages in ((0, FAKE, 0, 0), (FAKE, OFF, 0, 0), (FAKE, FAKE, FAKE, 0),
                  (FAKE, FAKE, FAKE, FAKE + 4)):
        assert call(pages=pages) == INVALID
    assert call(table=FAKE + 2) == call(starts=FAKE + 1) == INVALID


def test_append_at_arguments():
    assert _append_at(positions=None) == _append_at(positions=FAKE + 2) == INVALID
    assert _append_at(cos=None) == _append_at(rope=(0, 128, 0)) == _append_at(k=OFF) == INVALID
    assert _append_at(rope=(100, 120, 0)) == UNSUPPORTED


def test_draft_tree_arguments():
    call = _lib.load().spx_draft_tree
    assert call(None, 1, 4, FAKE, FAKE, None) == call(FAKE, 1, 4, None, FAKE, None) == INVALID
    assert call(FAKE, 1, 4, FAKE, None, None) == call(FAKE, 0, 4, FAKE, FAKE, None) == INVALID
    assert call(FAKE, 1, 0, FAKE, FAKE, None) == call(FAKE, 1, 257, FAKE, FAKE, None) == INVALID
    assert call(FAKE + 2, 1, 4, FAKE, FAKE, None) == call(FAKE, 1, 4, FAKE, FAKE + 4, None) == INVALID
    assert call(FAKE, (1 << 23) + 1, 4, FAKE, FAKE, None) == INVALID


def test_tree_attention_arguments():
    assert _tree(q=None) == _tree(q=OFF) == _tree(qs=ODD) == _tree(out=None) == _tree(out=OFF) == INVALID
    assert _tree(masks=None) == _tree(masks=FAKE + 4) == _tree(workspace=None) == INVALID
    assert _tree(q_heads=27) == _tree(max_keys=-1) == _tree(tokens=257) == INVALID
    assert _tree(batch=1 << 18, tokens=256, q_heads=32) == INVALID
    # units of 64 keys are counted in 32 bits
    assert _tree(width=1 << 23, batch=64) == INVALID and b"bad shape" in _lib.load().spx_last_error()
    size = _lib.load().spx_paged_tree_attention_workspace_bytes
    assert size(_cache(), 28, 0) > 0 and size(_cache(tokens=256), 28, 0) > size(_cache(), 28, 0)
    assert size(None, 28, 0) == size(_cache(), 27, 0) == size(_cache(), 28, -1) == -1
    assert size(_cache(dim=64), 28, 0) == size(_cache(tokens=257), 28, 0) == -1


def test_keep_path_arguments():
    assert _lib.load().spx_paged_keep_path(None, 1, *[None] * 8) == _keep(count=0) == INVALID
    for name in ("parents", "drafts", "targets", "accepted", "path_out", "following"):
        assert _keep(**{name: None}) == INVALID
    assert _keep(path_in=FAKE) == _keep(parents=None, drafts=None, targets=None) == INVALID
    given = dict(parents=None, drafts=None, targets=None, accepted=None, path_out=None, following=None)
    assert _keep(**given) == _keep(**given, path_in=FAKE + 2) == INVALID
    assert _keep(drafts=FAKE + 4) == _keep(following=FAKE + 4) == _keep(accepted=FAKE + 1) == INVALID
    assert _keep(tokens=257) == INVALID
    for other in (dict(page_size=64), dict(kv_heads=2), dict(tokens=2), dict(table=2 * FAKE), dict(held=3),
                  dict(pages=(FAKE,) * 4), dict(dim=256), dict(starts=2 * FAKE), dict(counts=FAKE)):
        assert _keep(caches=_cache() + _cache(**other), count=2) == INVALID
        assert b"cache 1" in _lib.load().spx_last_error()


def test_accumulate_weights_arguments():
    assert _weights(q=None) == _weights(q=OFF) == _weights(qs=ODD) == _weights(lse=None) == INVALID
    assert _weights(weights=None) == _weights(weights=FAKE + 2) == _weights(row=4095) == INVALID
    assert _weights(q_heads=27) == _weights(tokens=100, workspace=None) == INVALID
    assert _weights(tokens=100, workspace=OFF) == INVALID
    assert _weights(batch=1 << 16, tokens=1 << 10, q_heads=32) == INVALID
    assert _weights(width=1 << 23, batch=64, row=1 << 31) == INVALID
    size = _lib.load().spx_paged_accumulate_weights_workspace_bytes
    assert size(_cache(), 28) == 0 < size(_cache(tokens=100), 28)
    assert size(None, 28) == size(_cache(), 27) == -1


def test_evict_arguments():
    assert _evict(weights=None) == _evict(out=None) == _evict(positions_out=None) == INVALID
    assert _evict(lengths_out=None) == _evict(workspace=None) == _evict(workspace=FAKE + 4) == INVALID
    assert _evict(positions=FAKE + 2) == _evict(seen=FAKE + 2) == _evict(row=4095) == INVALID
    assert _evict(budget=0) == _evict(budget=-1) == _evict(recent=-1) == _evict(sinks=-1) == INVALID
    assert _evict(recent=99) == _evict(recent=2**31 - 1, sinks=2**31 - 1) == INVALID
    assert _evict(batch=1 << 20) == INVALID
    size = _lib.load().spx_paged_evict_workspace_bytes
    assert size(_cache(), 100) > 0 and size(_cache(), 0) == size(None, 100) == -1


def test_wrappers_refuse():
    """Tensors that are on no GPU."""
    cache = paged.empty_pages(4, 16, 2, 128, "cpu")
    x = torch.zeros(1, 3, 2, 128, dtype=torch.bfloat16)
    table, starts = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    parents, tokens = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int64)
    masks, lse, weights = tokens[..., None], torch.zeros(1, 3, 2), torch.zeros(1, 2, 64)
    rope = paged.rope_table(64, 128)
    for call in (lambda: paged.append_tokens(cache, table, starts, x, x, rope=rope, positions=parents),
                 lambda: paged.draft_tree(parents),
                 lambda: paged.tree_attention(x, cache, table, starts, masks, 0.1),
                 lambda: paged.accept_drafts(cache, table, starts, parents, tokens, tokens),
                 lambda: paged.keep_path([cache, cache], table, starts, parents),
                 lambda: paged.accumulate_weights(weights, x, lse, cache, table, starts, 0.1),
                 lambda: paged.evict_tokens(cache, table, starts, weights, 10),
                 lambda: _lib.host_module().draft_tree(parents, 0),
                 lambda: _lib.host_module().keep_path((cache,), table, starts, None, parents, 0),
                 lambda: _lib.host_module().evict(cache.key_pages, cache.value_pages, None, None, table,
                                                  starts, weights, None, None, 10, 0, 0, None, None, 0)):
        with pytest.raises(ValueError, match="ROCm GPU"):
            call()
    for call in (lambda: paged.draft_tree(None), lambda: paged.evict_tokens(cache, table, 3, weights, 10),
                 lambda: paged.keep_path(cache, table, starts, [0])):
        with pytest.raises(ValueError, match="expected a tensor"):
            call()


def test_description_size():
    """Several descriptions lie side by side as the C entry reads them."""
    assert len(_cache()) == 96 and ctypes.sizeof(ctypes.c_void_p) == 8


def test_keep_path_of_the_same_pages_twice():
    assert _keep(caches=_cache() + _cache(), count=2) == INVALID
    assert b"same pages" in _lib.load().spx_last_error()
