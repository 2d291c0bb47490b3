"""Paged KV cache on MI355X: append with the rotary embedding applied on the way, reading
back, and attention of new tokens over the pages, in bf16 or in 4 bits.

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
              the rest is padding

A new token is live if its sequence is not a free slot, it is no padding, and the table
reaches its position. Positions whose page id is outside the cache have no place: nothing is
stored for them and they are not seen. Nothing here reads these values on the host, so every
call can be captured in a HIP graph and replayed with other lengths. There is no derivative in
either mode: tensors that require a gradient are refused while gradients are recorded, and
those that carry a forward-mode tangent. The calls are refused while torch traces a graph
(``torch.jit.trace``, ``make_fx``, ``torch.export``); ``torch.compile`` breaks its graph at
them. q, k and v do not overlap the cache's memory, nor do its tensors each other's.
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


def _run(tensor: torch.Tensor, name: str, cache: PagedCache, *args):
    """A function of the host module on the tensor's device (the launch needs it to be the
    current one)."""
    if not isinstance(tensor, torch.Tensor):
        raise ValueError(f"expected a tensor, got {type(tensor).__name__}")
    if not tensor.is_cuda:
        _lib.require_gpu(tensor)
    device = tensor.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _run(tensor, name, cache, *args)
    return getattr(_lib.host_module(), name)(cache.key_pages, cache.value_pages, cache.key_scales,
                                             cache.value_scales, *args, _lib.stream_of(device))


def append_tokens(cache: PagedCache, page_table: torch.Tensor, starts: torch.Tensor,
                  k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None,
                  rope: tuple[torch.Tensor, torch.Tensor] | None = None,
                  counts: torch.Tensor | None = None, interleaved: bool = False,
                  return_keys: bool = False):
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
    sequence (full pages of a common prefix may be shared)."""
    cos, sin = rope if rope is not None else (None, None)
    return _run(k, "append", cache, page_table, starts, counts, k, v, q, cos, sin, interleaved,
                return_keys)


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
