"""Caches whose rows of an accepted path are moved: of memory that no two share."""

import pytest
import torch

from exp3_amd import paged

pytestmark = pytest.mark.gpu

PATH = torch.tensor([[0, 2, 3, -1]], dtype=torch.int32)


def _place():
    return (torch.arange(3, dtype=torch.int32, device="cuda")[None],
            torch.full((1,), 5, dtype=torch.int32, device="cuda"))


def test_caches_that_share_memory_are_refused(gpu):
    pool = torch.randn(20, 2, 16, 128, device="cuda").to(torch.bfloat16)
    before = pool.clone()
    k, v, other = pool[:4], pool[4:8], paged.PagedCache(pool[8:12], pool[12:16])
    place = _place()
    for caches in ((paged.PagedCache(k, k),), (paged.PagedCache(k, v), paged.PagedCache(v, k)),
                   (paged.PagedCache(k, v), other, paged.PagedCache(pool[16:], pool[7:11])),
                   (paged.PagedCache(pool[3:7], pool[7:11]), other),
                   [paged.PagedCache(k, v)] * 2):
        with pytest.raises(ValueError, match="overlap|same pages"):
            paged.keep_path(caches, *place, PATH.cuda())
        with pytest.raises(ValueError, match="overlap|same pages"):
            paged.accept_drafts(caches, *place, PATH.cuda(), PATH.cuda().long(), PATH.cuda().long())
    torch.cuda.synchronize()
    assert torch.equal(pool, before)
    bytes_ = torch.randint(100, 140, (4, 4, 2, 16, 64), dtype=torch.uint8, device="cuda")
    scales = torch.randint(120, 124, (4, 2, 16, 4), dtype=torch.uint8, device="cuda")
    first, second = (paged.PagedCache(bytes_[2 * i], bytes_[2 * i + 1], scales, scales.clone())
                     for i in range(2))
    with pytest.raises(ValueError, match="overlap"):
        paged.keep_path((first, second), *place, PATH.cuda())


def test_caches_side_by_side(gpu):
    """All layers in one tensor, in any order."""
    pool = torch.randn(6, 4, 2, 16, 128, device="cuda").to(torch.bfloat16)
    want = pool.transpose(2, 3).clone()                           # [.., page, slot, Hkv, D]
    for to, of in ((6, 7), (7, 8)):
        want[:, 0, to] = want[:, 0, of]
    caches = [paged.PagedCache(pool[i], pool[j]) for i, j in ((5, 0), (2, 1), (3, 4))]
    paged.keep_path(caches, *_place(), PATH.cuda())
    assert torch.equal(pool, want.transpose(2, 3))
