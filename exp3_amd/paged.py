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
from functools import lru_cache
import struct

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


# spx_paged_cache of the C header, and the strides of a [B, T, H, D] tensor
_DESCRIPTION = struct.Struct("7Pq8i")
_STRIDES = struct.Struct("4q")
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _check_cache(cache: PagedCache, device: int) -> tuple:
    """(four pointers), pages, page_size, kv_heads, head_dim of a cache on this device index."""
    key, value, key_scales, value_scales = (cache.key_pages, cache.value_pages, cache.key_scales,
                                            cache.value_scales)
    shape = key.shape
    dtype = torch.bfloat16 if key_scales is None else torch.uint8
    if not (len(shape) == 4 and value.shape == shape and key.dtype is dtype and value.dtype is dtype
            and key.is_contiguous() and value.is_contiguous()):
        raise ValueError(f"pages must be contiguous {dtype} [pages, Hkv, page_size, "
                         f"{'D' if key_scales is None else 'D // 2'}] tensors of one shape, got "
                         f"{tuple(shape)} {key.dtype} and {tuple(value.shape)} {value.dtype}")
    if not key.get_device() == value.get_device() == device:
        raise ValueError(f"pages on {key.device} and {value.device}, the call's tensors on device "
                         f"{device}")
    pages, kv_heads, page_size, width = shape
    if key_scales is None:
        if value_scales is not None:
            raise ValueError("a 4-bit cache needs key_scales and value_scales, a bf16 cache neither")
        return (key.data_ptr(), value.data_ptr(), 0, 0), pages, page_size, kv_heads, width
    if value_scales is None:
        raise ValueError("a 4-bit cache needs key_scales and value_scales, a bf16 cache neither")
    groups = (pages, kv_heads, page_size, 2 * width // SCALE_GROUP)
    for x in (key_scales, value_scales):
        if not (x.shape == groups and x.dtype is torch.uint8 and x.is_contiguous()
                and x.get_device() == device):
            raise ValueError(f"scales must be contiguous uint8 {groups} on the pages' device, got "
                             f"{tuple(x.shape)} {x.dtype} on {x.device}")
    return (key.data_ptr(), value.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr()), \
        pages, page_size, kv_heads, 2 * width


def _lengths(name: str, x: torch.Tensor, batch: int, device: int) -> int:
    if not (x.dtype is torch.int32 and x.shape == (batch,) and x.get_device() == device
            and x.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 [{batch}] tensor on the pages' device, "
                         f"got {tuple(x.shape)} {x.dtype} on {x.device}")
    return x.data_ptr()


def _describe(cache: PagedCache, page_table, starts, counts, batch: int, tokens: int,
              device: int) -> tuple[bytes, int, int, tuple]:
    """The C description of a call's cache and tokens, checked, its kv_heads and head_dim, and
    what the size of a workspace depends on."""
    pointers, pages, page_size, kv_heads, head_dim = _check_cache(cache, device)
    shape = page_table.shape
    if not (page_table.dtype is torch.int32 and len(shape) == 2 and shape[0] == batch
            and page_table.get_device() == device):
        raise ValueError(f"page_table must be an int32 [{batch}, pages per sequence] tensor on the "
                         f"pages' device, got {tuple(shape)} {page_table.dtype} on "
                         f"{page_table.device}")
    row, unit = page_table.stride()
    if unit != 1 and shape[1] > 1:
        raise ValueError("page_table must have unit stride within a row")
    sizes = (shape[1], pages, page_size, kv_heads, head_dim, batch, tokens, 0)
    return _DESCRIPTION.pack(*pointers, page_table.data_ptr(),
                             _lengths("starts", starts, batch, device),
                             0 if counts is None else _lengths("counts", counts, batch, device),
                             row, *sizes), kv_heads, head_dim, sizes


def _rows(x: torch.Tensor) -> torch.Tensor:
    """A [B, T, H, D] bf16 tensor that the kernels read in place."""
    return _lib.kernel_view(x.resolve_neg() if x.is_neg() else x)


def _new_rows(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _call(device: int, name: str, *args) -> None:
    """Enqueue on the tensors' device (the launch needs it to be the current one)."""
    if device == _current_device():
        _lib.call(name, *args, _lib.stream_of(device))
        return
    with torch.cuda.device(device):
        _lib.call(name, *args, _lib.stream_of(device))


@lru_cache(maxsize=256)
def _workspace_bytes(four_bit: bool, sizes: tuple, q_heads: int, max_keys: int) -> int:
    mark = 16 if four_bit else 0
    return _lib.load().spx_paged_attention_workspace_bytes(
        _DESCRIPTION.pack(16, 16, mark, mark, 16, 16, 0, 0, *sizes), q_heads, max_keys)


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
    device = _lib.require_gpu(k, v, q).index
    k, v = _rows(k), _rows(v)
    shape = k.shape
    if shape != v.shape:
        raise ValueError(f"k {tuple(shape)} and v {tuple(v.shape)} differ")
    batch, tokens, kv_heads, head_dim = shape
    place, held_heads, held_dim, _ = _describe(cache, page_table, starts, counts, batch, tokens,
                                               device)
    if kv_heads != held_heads or head_dim != held_dim:
        raise ValueError(f"k {tuple(shape)} does not fit a cache of {held_heads} heads of {held_dim}")
    q_part, q_heads, q_out = (None, None), 0, None
    if q is not None:
        q = _rows(q)
        q_heads = q.shape[2]
        if q.shape != (batch, tokens, q_heads, head_dim) or q_heads == 0:
            raise ValueError(f"q {tuple(q.shape)} does not match k {tuple(shape)}")
        q_out = _new_rows(q)
        q_part = (q.data_ptr(), _STRIDES.pack(*q.stride()))
    k_out = _new_rows(k) if return_keys else None
    table = (None, None, 0, 0)
    if rope is not None:
        cos, sin = rope
        if not (cos.dtype is torch.float32 and sin.dtype is torch.float32 and cos.dim() == 2
                and sin.shape == cos.shape and cos.is_contiguous() and sin.is_contiguous()
                and cos.get_device() == sin.get_device() == device):
            raise ValueError("rope must be two contiguous float32 [positions, rotary_dim // 2] "
                             "tensors of one shape on the pages' device")
        positions, half = cos.shape
        table = (cos.data_ptr(), sin.data_ptr(), positions, 2 * half)
    if batch and tokens:
        _call(device, "spx_paged_append", place, *q_part, k.data_ptr(), _STRIDES.pack(*k.stride()),
              v.data_ptr(), _STRIDES.pack(*v.stride()), q_heads, *table, int(interleaved),
              _lib.ptr(q_out), _lib.ptr(k_out))
    return q_out, k_out


def gather_tokens(cache: PagedCache, page_table: torch.Tensor, starts: torch.Tensor, tokens: int,
                  counts: torch.Tensor | None = None):
    """K and V of positions ``starts[b] .. starts[b] + tokens`` as contiguous bf16
    ``[B, tokens, Hkv, D]`` (4-bit values are exact in bf16); rows that are not live or have no
    place are 0."""
    device = _lib.require_gpu(cache.key_pages, page_table).index
    if tokens < 0:
        raise ValueError(f"tokens must not be negative, got {tokens}")
    batch = page_table.shape[0]
    place, kv_heads, head_dim, _ = _describe(cache, page_table, starts, counts, batch, tokens, device)
    shape = (batch, tokens, kv_heads, head_dim)
    k = cache.key_pages.new_empty(shape, dtype=torch.bfloat16)
    v = cache.key_pages.new_empty(shape, dtype=torch.bfloat16)
    if batch and tokens:
        _call(device, "spx_paged_gather", place, k.data_ptr(), v.data_ptr())
    return k, v


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
    device = _lib.require_gpu(q, cache.key_pages).index
    q = _rows(q)
    shape = q.shape
    batch, tokens, q_heads, head_dim = shape
    place, kv_heads, held_dim, sizes = _describe(cache, page_table, starts, counts, batch, tokens,
                                                 device)
    if head_dim != held_dim or q_heads == 0 or kv_heads == 0 or q_heads % kv_heads:
        raise ValueError(f"q {tuple(shape)} does not fit a cache of {kv_heads} heads of {held_dim}")
    bound = 0 if max_keys is None else int(max_keys)
    if bound < 0:
        raise ValueError(f"max_keys must not be negative, got {max_keys}")
    out = _new_rows(q)
    lse = q.new_empty(shape[:3], dtype=torch.float32) if return_lse else None
    if batch and tokens:
        nbytes = _workspace_bytes(cache.key_scales is not None, sizes, q_heads, bound)
        workspace = q.new_empty(nbytes, dtype=torch.uint8) if nbytes > 0 else None
        _call(device, "spx_paged_attention", place, q.data_ptr(), _STRIDES.pack(*q.stride()), q_heads,
              bound, float(scale), _lib.ptr(workspace), out.data_ptr(), _lib.ptr(lse))
    return (out, lse) if return_lse else out
