"""Paged KV cache on MI355X: append with the rotary embedding applied on the way, reading
back, attention of new tokens over the pages, in bf16 or in 4 bits, drafted trees, and eviction of
the tokens that gathered least attention.

The serving side of the prefill backend: a prompt's projections go through
``append_tokens`` (which stores K and V and returns the rotated Q and K that
``attention.AttentionBackend`` takes for the prefill), and every later step appends its
tokens and calls ``paged_attention``. So does a chunk of a prompt behind a cached prefix: the
backend takes fewer queries than keys for a decode step and applies no mask. The reference
keeps its cache in transformers' DynamicCache (evaluate.py) and has no counterpart of these
functions.

Common arguments:

  cache       PagedCache, e.g. from ``empty_pages``
  page_table  int32 [B, W] on the GPU: page ids of each sequence; position p of sequence b
              is slot ``p % page_size`` of page ``page_table[b, p // page_size]``
  starts      int32 [B]: the position of each sequence's first new token, i.e. the tokens
              held before; negative for a free slot of the batch
  counts      int32 [B] or None: how many of the T new tokens of each sequence are tokens;
              the rest is padding, whose rows may hold anything

A new token is live if its sequence is not a free slot, it is no padding, and the table
reaches its position. Positions whose page id is outside the cache have no place: nothing is
stored for them and they are not seen. Nothing here reads these values on the host, so every
call can be captured in a HIP graph and replayed with other lengths. There is no derivative in
either mode: tensors that require a gradient are refused while gradients are recorded, and
those that carry a forward-mode tangent. The calls are refused while torch traces a graph
(``torch.jit.trace``, ``make_fx``, ``torch.export``); ``torch.compile`` breaks its graph at
them. q, k and v do not overlap the cache's memory, nor do its tensors each other's.

A step of a drafted tree is ``draft_tree`` once, per layer ``append_tokens`` (with ``positions =
starts[:, None] + depths``) and ``tree_attention``, and ``accept_drafts`` once for all layers. A cache
held at a budget takes ``accumulate_weights`` behind the attention calls (with ``return_lse``) and now and
then ``evict_tokens``.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib

MIN_PAGE, MAX_PAGE = 16, 1024
SCALE_GROUP = 32        # dims per scale of a 4-bit page


@dataclass
class PagedCache:
    """``key_pages`` / ``value_pages``: bf16 ``[pages, Hkv, page_size, D]``; or, with scales
    given, 4 bits: uint8 ``[pages, Hkv, page_size, D // 2]`` (E2M1 values, the even dim in the
    low half) with uint8 scales ``[pages, Hkv, page_size, D // 32]`` (E8M0: 2^(byte - 127),
    255 is NaN), the microscaling format MXFP4."""
    key_pages: torch.Tensor
    value_pages: torch.Tensor
    key_scales: torch.Tensor | None = None
    value_scales: torch.Tensor | None = None

    @property
    def four_bit(self) -> bool:
        return self.key_scales is not None

    @property
    def page_size(self) -> int:
        return self.key_pages.shape[2]

    @property
    def kv_heads(self) -> int:
        return self.key_pages.shape[1]

    @property
    def head_dim(self) -> int:
        return self.key_pages.shape[3] * (2 if self.four_bit else 1)


def empty_pages(pages: int, page_size: int, kv_heads: int, head_dim: int, device,
                four_bit: bool = False) -> PagedCache:
    """An uninitialised cache: pages are read only where tokens have been appended."""
    if head_dim not in (128, 256):
        raise ValueError(f"head_dim {head_dim} unsupported (128 or 256)")
    if not MIN_PAGE <= page_size <= MAX_PAGE or page_size & (page_size - 1):
        raise ValueError(f"page_size {page_size} unsupported (a power of two from {MIN_PAGE} to "
                         f"{MAX_PAGE})")
    shape = (pages, kv_heads, page_size)

    def empty(last, dtype):
        return torch.empty(*shape, last, dtype=dtype, device=device)

    if not four_bit:
        return PagedCache(empty(head_dim, torch.bfloat16), empty(head_dim, torch.bfloat16))
    half, groups = head_dim // 2, head_dim // SCALE_GROUP
    return PagedCache(empty(half, torch.uint8), empty(half, torch.uint8),
                      empty(groups, torch.uint8), empty(groups, torch.uint8))


def rope_table(positions: int, rotary_dim: int, theta: float = 1.0e6, device=None):
    """fp32 (cos, sin) ``[positions, rotary_dim // 2]``, the angles formed in fp64 (in fp32
    those of positions near 131072 are off by up to 2^-8)."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} must be even and positive")
    inv = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _run(tensor: torch.Tensor, name: str, cache: PagedCache | None, *args, more=()):
    """A function of the host module on the tensor's device (the launch needs it to be the
    current one)."""
    if not isinstance(tensor, torch.Tensor):
        raise ValueError(f"expected a tensor, got {type(tensor).__name__}")
    if not tensor.is_cuda:
        _lib.require_gpu(tensor)
    device = tensor.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _run(tensor, name, cache, *args, more=more)
    call = getattr(_lib.host_module(), name)
    if cache is None:
        return call(*args, _lib.stream_of(device))
    return call(cache.key_pages, cache.value_pages, cache.key_scales, cache.value_scales, *args,
                _lib.stream_of(device), *more)


def append_tokens(cache: PagedCache, page_table: torch.Tensor, starts: torch.Tensor,
                  k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None,
                  rope: tuple[torch.Tensor, torch.Tensor] | None = None,
                  counts: torch.Tensor | None = None, interleaved: bool = False,
                  return_keys: bool = False, positions: torch.Tensor | None = None):
    """Rotate ``k`` (and ``q``), store ``k`` and ``v`` -> (rotated q or None, rotated k or None).

    k, v: bf16 ``[B, T, Hkv, D]``, q: bf16 ``[B, T, Hq, D]``, any strides (slices of one fused
    projection are read in place); with ``return_keys`` the rotated keys come back too, as a
    prefill needs them. ``rope``: fp32 (cos, sin) ``[positions, rotary_dim // 2]`` reaching as
    far as the page table, e.g. ``rope_table``; the first ``rotary_dim`` dims are rotated,
    paired by halves (or neighbours, ``interleaved``). bf16 rows are rotated in fp32 and
    rounded once. 4-bit rows are rounded to nearest (ties to the even code) from the rotated
    value itself; the scale of 32 dims is the power of two that puts the largest into
    [3.5, 7), values above 6 become 6, and 32 dims with one that is not finite read back
    as NaN. Returned rows of tokens that are not live are 0.

    Two tokens of a call must not have the same place: pages that are appended to belong to one
    sequence (full pages of a common prefix may be shared).

    ``positions``: int32 ``[B, T]``, the tokens' positions in the text for the rotation where they
    are not their places in the cache: ``starts[:, None] + depths`` for the nodes of a drafted tree,
    those of the text behind an eviction. ``rope`` then reaches as far as the text; dims that it
    does not reach are stored and returned as NaN."""
    cos, sin = rope if rope is not None else (None, None)
    more = () if positions is None else (positions,)
    return _run(k, "append", cache, page_table, starts, counts, k, v, q, cos, sin, interleaved,
                return_keys, more=more)


def gather_tokens(cache: PagedCache, page_table: torch.Tensor, starts: torch.Tensor, tokens: int,
                  counts: torch.Tensor | None = None):
    """K and V of positions ``starts[b] .. starts[b] + tokens`` as contiguous bf16
    ``[B, tokens, Hkv, D]`` (4-bit values are exact in bf16); rows that are not live or have no
    place are 0."""
    return _run(page_table, "gather", cache, page_table, starts, counts, tokens)


def paged_attention(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor,
                    starts: torch.Tensor, scale: float, counts: torch.Tensor | None = None,
                    max_keys: int | None = None, return_lse: bool = False):
    """softmax(scale q K^T) V of new tokens over the cache that already holds them.

    q: bf16 ``[B, T, Hq, D]`` (rotated); token i of sequence b sees positions
    ``0 .. starts[b] + i`` -> bf16 ``[B, T, Hq, D]``, with ``return_lse`` also the natural-log
    LSE, fp32 ``[B, T, Hq]``. Tokens that are not live, see nothing, or have no score above -inf
    give 0 and -inf. ``max_keys``: an upper bound of ``starts[b] + T`` where the caller has one;
    it only chooses how the work is divided, and pays where the table reaches far and all
    sequences are short (up to 512 keys, 1024 in 4 bits at D = 128). Meant for decode steps and
    a few drafted tokens: each 16 of the T x Hq / Hkv rows of a KV head read K and V anew."""
    return _run(q, "attention", cache, page_table, starts, counts, q, scale,
                0 if max_keys is None else max_keys, return_lse)


# ------------------------------------------------------------- drafted trees

def draft_tree(parents: torch.Tensor):
    """The plan of trees of drafted tokens -> (depths int32 ``[B, T]``, masks int64
    ``[B, T, ceil(T / 64)]``).

    parents: int32 ``[B, T]``, T at most 256: the node that each one follows, one before it; any
    other value (-1) for nodes that follow the cached tokens. ``masks``: bit ``j % 64`` of word
    ``j // 64`` of row i is set where j is i or one of its ancestors; ``depths``: how many ancestors
    a node has. Made once for a step, used by all layers."""
    return _run(parents, "draft_tree", None, parents)


def tree_attention(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor,
                   starts: torch.Tensor, masks: torch.Tensor, scale: float,
                   counts: torch.Tensor | None = None, max_keys: int | None = None,
                   return_lse: bool = False):
    """Attention of a tree of drafted tokens over the cache that already holds them: as
    ``paged_attention``, but node i of sequence b (in place ``starts[b] + i``) sees the places below
    ``starts[b]`` and the live nodes j whose bit is set in row i of ``masks``, e.g. from
    ``draft_tree`` (any bits may be set). At most 256 nodes; K and V are read once for each 128 of
    the T x Hq / Hkv rows of a KV head. ``max_keys``: an upper bound of ``starts[b] + T``, which only
    chooses how the work is divided."""
    return _run(q, "tree_attention", cache, page_table, starts, counts, q, masks, scale,
                0 if max_keys is None else max_keys, return_lse)


def _caches(caches):
    return (caches,) if isinstance(caches, PagedCache) else tuple(caches)


def accept_drafts(caches, page_table: torch.Tensor, starts: torch.Tensor, parents: torch.Tensor,
                  drafts: torch.Tensor, targets: torch.Tensor, counts: torch.Tensor | None = None):
    """The drafts that the model agrees with, moved into place in every cache -> (accepted int32
    ``[B]``, path int32 ``[B, T]``, following int64 ``[B]``).

    caches: a PagedCache or those of all layers, alike but for their pages, which share no memory (those
    of the drafts' rows belong to one sequence). parents: as ``draft_tree``; drafts, targets: int64 ``[B, T]``, a node's token and the token that the model
    chose behind it. Node 0 (the last token that was decided) is accepted, then the first child whose
    draft is the target of the node accepted last, as long as there is one. ``path``: the accepted
    nodes, then -1; ``following``: the target of the last one, the next token. K and V of the
    accepted nodes move to ``starts[b] .. starts[b] + accepted[b]``. No live node: 0 and -1."""
    return _run(parents, "keep_path", None, _caches(caches), page_table, starts, counts, parents,
                drafts, targets)


def keep_path(caches, page_table: torch.Tensor, starts: torch.Tensor, path: torch.Tensor,
              counts: torch.Tensor | None = None) -> None:
    """K and V of a path that the caller accepted moved into place, in every cache: those of
    ``starts[b] + path[b, j]`` to ``starts[b] + j``. path: int32 ``[B, T]``, T at most 256, live nodes
    that ascend; it ends at the first one that is not one (-1)."""
    _run(path, "keep_path", None, _caches(caches), page_table, starts, counts, path)


# ------------------------------------------------------------------ eviction

def accumulate_weights(weights: torch.Tensor, q: torch.Tensor, lse: torch.Tensor, cache: PagedCache,
                       page_table: torch.Tensor, starts: torch.Tensor, scale: float,
                       counts: torch.Tensor | None = None) -> None:
    """Add the attention weight that cached tokens receive from new ones, in place.

    weights: fp32 ``[B, Hkv, slots]``, at least as many slots as the page table reaches, 0 where a
    sequence begins; q and the other arguments as given to ``paged_attention``, lse: what it returned
    with ``return_lse``. ``weights[b, kvh, p]`` grows by the sum over the rows (tokens, query heads of
    the KV head) that see position p of their probability for it. Rows that see nothing add nothing.
    A prompt's tokens are judged by its last ones: ``starts`` the prompt's length less T, q the
    rotated queries of its last T tokens. Reads K once, whatever T."""
    _run(q, "accumulate", cache, page_table, starts, counts, weights, q, lse, scale)


def evict_tokens(cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor,
                 weights: torch.Tensor, budget: int, positions: torch.Tensor | None = None,
                 seen: torch.Tensor | None = None, recent: int = 0, sinks: int = 0,
                 out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Drop the tokens of each KV head that gathered least, down to ``budget`` -> (lengths, weights,
    positions).

    lengths: int32 ``[B]``, tokens held (negative: a free slot). Kept are those whose position in the
    text is below ``sinks`` or among the last ``recent`` (together at most ``budget``), then those of
    the largest weight, the lower slot first among equals; NaN counts least. Heads keep different
    tokens: the cache's slots are no positions any more. Tokens kept below slot ``budget`` stay, the
    freed slots are filled in order with the ones kept behind it, so little moves and every later
    append goes to the new end.

    positions: int32, as weights, -1 for tokens appended since (all of them: None): those have
    position ``seen[b] - lengths[b] + slot``; seen: int32 ``[B]``, tokens of the text so far (None:
    the lengths, right for the first eviction). Returned are the new lengths and the new ``weights``
    and ``positions`` (0 and -1 behind the end), in ``out`` if given: the tensors themselves, or
    others that share no memory with an argument. Sequences within the budget, or with a token that has no place, keep all. Later
    tokens are appended with ``positions=``. Pages that are written to belong to one sequence."""
    return _run(lengths, "evict", cache, page_table, lengths, weights, positions, seen, budget,
                recent, sinks, *(out if out is not None else (None, None)))
