"""Paged KV cache on MI355X: append with the rotary embedding applied on the way, reading
back, and attention of new tokens over the pages, in bf16 or in 4 bits.

The serving side of the prefill backend: a prompt's projections go through
``append_tokens`` (which stores K and V and returns the rotated Q and K that
``attention.AttentionBackend`` takes for the prefill), and every later step appends its
tokens and calls ``paged_attention``. The reference keeps its cache in transformers'
DynamicCache (evaluate.py) and has no counterpart of these functions.

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
call can be captured in a HIP graph and replayed with other lengths. There is no backward
pass.
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
    inv = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _check_cache(cache: PagedCache, device: torch.device) -> tuple:
    """The cache's part of a call's arguments, checked: (four pointers, pages, page_size),
    kv_heads, head_dim."""
    key, value, key_scales, value_scales = (cache.key_pages, cache.value_pages, cache.key_scales,
                                            cache.value_scales)
    four = key_scales is not None
    if four != (value_scales is not None):
        raise ValueError("a 4-bit cache needs key_scales and value_scales, a bf16 cache neither")
    shape = key.shape
    dtype = torch.uint8 if four else torch.bfloat16
    if len(shape) != 4 or value.shape != shape or key.dtype != dtype or value.dtype != dtype \
            or not key.is_contiguous() or not value.is_contiguous():
        raise ValueError(f"pages must be contiguous {dtype} [pages, Hkv, page_size, D"
                         f"{' // 2' if four else ''}] tensors of one shape, got {tuple(shape)} "
                         f"{key.dtype} and {tuple(value.shape)} {value.dtype}")
    pages, kv_heads, page_size, width = shape
    head_dim = 2 * width if four else width
    if four:
        groups = (pages, kv_heads, page_size, head_dim // SCALE_GROUP)
        for s in (key_scales, value_scales):
            if s.shape != groups or s.dtype != torch.uint8 or not s.is_contiguous():
                raise ValueError(f"scales must be contiguous uint8 {groups}, got "
                                 f"{tuple(s.shape)} {s.dtype}")
            if s.device != device:
                raise ValueError(f"tensors on different devices: {device} and {s.device}")
    for x in (key, value):
        if x.device != device:
            raise ValueError(f"tensors on different devices: {device} and {x.device}")
    return (key.data_ptr(), value.data_ptr(), _lib.ptr(key_scales), _lib.ptr(value_scales), pages,
            page_size), kv_heads, head_dim


def _check_map(page_table, starts, counts, batch: int, device: torch.device) -> tuple:
    """(table, its stride, its width, starts, counts) as the entry points take them."""
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != batch:
        raise ValueError(f"page_table must be int32 [{batch}, pages per sequence], got "
                         f"{tuple(page_table.shape)} {page_table.dtype}")
    for name, x in (("starts", starts), ("counts", counts)):
        if x is None:
            continue
        if x.dtype != torch.int32 or x.shape != (batch,):
            raise ValueError(f"{name} must be int32 [{batch}], got {tuple(x.shape)} {x.dtype}")
        if x.device != device:
            raise ValueError(f"tensors on different devices: {device} and {x.device}")
        if x.stride(0) != 1 and batch > 1:
            raise ValueError(f"{name} must be contiguous")
    if page_table.device != device:
        raise ValueError(f"tensors on different devices: {device} and {page_table.device}")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table must have unit stride within a row")
    return (page_table.data_ptr(), page_table.stride(0), page_table.shape[1], starts.data_ptr(),
            _lib.ptr(counts))


def _rows(x: torch.Tensor) -> torch.Tensor:
    """A [B, T, H, D] bf16 tensor that the kernels read in place."""
    return _lib.kernel_view(x.resolve_neg() if x.is_neg() else x)


def _call(device: torch.device, name: str, *args) -> None:
    """Enqueue on the tensors' device (the launch needs it to be the current one)."""
    if device.index == torch.cuda.current_device():
        _lib.call(name, *args, _lib.stream(device))
        return
    with torch.cuda.device(device):
        _lib.call(name, *args, _lib.stream(device))


@torch.no_grad()
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
    device = _lib.require_gpu(k, v, q)
    k, v = _rows(k), _rows(v)
    if k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    batch, tokens, kv_heads, head_dim = k.shape
    pages, held_heads, held_dim = _check_cache(cache, device)
    if (kv_heads, head_dim) != (held_heads, held_dim):
        raise ValueError(f"k {tuple(k.shape)} does not fit a cache of {held_heads} heads of "
                         f"{held_dim}")
    place = _check_map(page_table, starts, counts, batch, device)
    q_heads, q_out = 0, None
    if q is not None:
        q = _rows(q)
        q_heads = q.shape[2]
        if q.shape != (batch, tokens, q_heads, head_dim) or q_heads == 0:
            raise ValueError(f"q {tuple(q.shape)} does not match k {tuple(k.shape)}")
        q_out = torch.empty(q.shape, dtype=torch.bfloat16, device=device)
    k_out = torch.empty(k.shape, dtype=torch.bfloat16, device=device) if return_keys else None
    table = (None, None, 0, 0)
    if rope is not None:
        cos, sin = rope
        for x in rope:
            if x.dtype != torch.float32 or x.dim() != 2 or x.shape != cos.shape \
                    or not x.is_contiguous():
                raise ValueError("rope must be two contiguous float32 [positions, rotary_dim // 2] "
                                 "tensors of one shape")
            if x.device != device:
                raise ValueError(f"tensors on different devices: {device} and {x.device}")
        table = (cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1])
    if batch and tokens:
        _call(device, "spx_paged_append", _lib.ptr(q), _lib.strides(q), k.data_ptr(),
              _lib.strides(k), v.data_ptr(), _lib.strides(v), *table, int(interleaved), *place,
              *pages, batch, tokens, q_heads, kv_heads, head_dim, _lib.ptr(q_out), _lib.ptr(k_out))
    return q_out, k_out


@torch.no_grad()
def gather_tokens(cache: PagedCache, page_table: torch.Tensor, starts: torch.Tensor, tokens: int,
                  counts: torch.Tensor | None = None):
    """K and V of positions ``starts[b] .. starts[b] + tokens`` as contiguous bf16
    ``[B, tokens, Hkv, D]`` (4-bit values are exact in bf16); rows that are not live or have no
    place are 0."""
    device = _lib.require_gpu(cache.key_pages, page_table)
    pages, kv_heads, head_dim = _check_cache(cache, device)
    batch = page_table.shape[0]
    place = _check_map(page_table, starts, counts, batch, device)
    if tokens < 0:
        raise ValueError(f"tokens must not be negative, got {tokens}")
    k = torch.empty(batch, tokens, kv_heads, head_dim, dtype=torch.bfloat16, device=device)
    v = torch.empty_like(k)
    if batch and tokens:
        _call(device, "spx_paged_gather", *place, *pages, batch, tokens, kv_heads, head_dim,
              k.data_ptr(), v.data_ptr())
    return k, v


@torch.no_grad()
def paged_attention(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor,
                    starts: torch.Tensor, scale: float, counts: torch.Tensor | None = None,
                    max_keys: int | None = None, return_lse: bool = False):
    """softmax(scale q K^T) V of new tokens over the cache that already holds them.

    q: bf16 ``[B, T, Hq, D]`` (rotated); token i of sequence b sees positions
    ``0 .. starts[b] + i`` -> bf16 ``[B, T, Hq, D]``, with ``return_lse`` also the natural-log
    LSE, fp32 ``[B, T, Hq]``. Tokens that are not live, or see nothing, give 0 and -inf.
    ``max_keys``: an upper bound of ``starts[b] + T`` where the caller has one; it only chooses
    how the work is divided. Meant for decode steps and a few drafted tokens: each 16 of the
    T x Hq / Hkv rows of a KV head read K and V anew."""
    device = _lib.require_gpu(q, cache.key_pages)
    q = _rows(q)
    batch, tokens, q_heads, head_dim = q.shape
    pages, kv_heads, held_dim = _check_cache(cache, device)
    if head_dim != held_dim or q_heads == 0 or kv_heads == 0 or q_heads % kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {kv_heads} heads of {held_dim}")
    place = _check_map(page_table, starts, counts, batch, device)
    bound = 0 if max_keys is None else max_keys
    if bound < 0:
        raise ValueError(f"max_keys must not be negative, got {max_keys}")
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=device) if return_lse else None
    if batch and tokens:
        shape = (batch, tokens, q_heads, kv_heads, head_dim)
        nbytes = _lib.load().spx_paged_attention_workspace_bytes(
            place[2], pages[5], bound, cache.four_bit, *shape)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None
        _call(device, "spx_paged_attention", q.data_ptr(), _lib.strides(q), *place, *pages, bound,
              *shape, float(scale), _lib.ptr(workspace), out.data_ptr(), _lib.ptr(lse))
    return (out, lse) if return_lse else out
