// Paged KV cache shared by the append, gather and attention kernels.
//
// Pages: [pages, Hkv, page_size, D] bf16, or in 4 bits [pages, Hkv, page_size, D / 2] bytes
// (E2M1, even dim in the low half) with scales [pages, Hkv, page_size, D / 32] (E8M0). A
// (page, head) pair is one contiguous run of rows, so 16 consecutive tokens of a head are one
// run of 4 KB (bf16, D = 128) or 1 KB + 64 bytes (4 bits).
#pragma once

#include "common.h"

namespace spx {

constexpr int kPagedGroup = 32;          // dims per scale of a 4-bit page
constexpr int kPagedMinPage = 16, kPagedMaxPage = 1024;

// Device data that no kernel of the stream writes meanwhile, at a uniform address.
__device__ __forceinline__ int scalar_load(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
}

// Which tokens a call is about and where they are: token i of sequence b has position
// starts[b] + i and is live if starts[b] >= 0, i < counts[b] (counts may be null) and the
// position is within the table.
struct PagedMap {
  const int32_t* table;                  // [B, width], rows table_stride apart
  int64_t table_stride;
  const int32_t* starts;
  const int32_t* counts;
  int width, pages, page_shift, kv_heads;

  __device__ __forceinline__ int64_t capacity() const { return (int64_t)width << page_shift; }
  // Position of token i of sequence b, or -1; b and i are uniform.
  __device__ __forceinline__ int position(int b, int i) const {
    const int start = scalar_load(starts + b);
    const int count = counts != nullptr ? scalar_load(counts + b) : i + 1;
    const int64_t p = (int64_t)start + i;
    return start >= 0 && i < count && p < capacity() ? (int)p : -1;
  }
  // Page of a position, the same for all lanes, or -1 also for position -1.
  __device__ __forceinline__ int uniform_page(int b, int p) const {
    const int id = scalar_load(table + b * table_stride + (max(p, 0) >> page_shift));
    return p >= 0 && (unsigned)id < (unsigned)pages ? id : -1;
  }
  // Page of a position, or -1 where the table names none, also for position -1 (the last one of a
  // sequence without keys), which reads nothing in front of the table.
  __host__ __device__ __forceinline__ int page(int b, int p) const {
    const int id = table[b * table_stride + ((p > 0 ? p : 0) >> page_shift)] | p >> 31;
    return (unsigned)id < (unsigned)pages ? id : -1;
  }
  // Row (of D elements) of a position of a KV head in the page arrays.
  __device__ __forceinline__ int64_t row(int page_id, int head, int p) const {
    return (((int64_t)page_id * kv_heads + head) << page_shift) + (p & ((1 << page_shift) - 1));
  }
};

// Eight 4-bit values as bf16: exact, a value has two bits.
__device__ __forceinline__ u32x4 widen8(uint32_t w, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
}

// Checks of a cache description; fills the map.
int paged_map(PagedMap& m, const spx_paged_cache* cache);

}  // namespace spx
