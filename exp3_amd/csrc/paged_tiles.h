// Rows of the paged cache as matrix operands, and the division of work over a grid: what the
// attention and weight kernels of the paged cache share.
#pragma once

#include "paged.h"

namespace spx {

__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

__device__ __forceinline__ int first_lane(int x) { return __builtin_amdgcn_readfirstlane(x); }

// n / d for n >= 0, inv = 1.0 / d: the quotient is off by one at most before it is put right. (An
// integer division takes some 40 dependent instructions.)
__device__ __forceinline__ int divide(int n, int d, double inv) {
  const int q = (int)((double)n * inv);
  const int r = n - q * d;
  return q + (r >= d ? 1 : 0) - (r < 0 ? 1 : 0);
}

// Sum over the lanes up to this one.
__device__ __forceinline__ int wave_prefix(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);    // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);    // row_bcast 15, 31
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

// Page memory as global memory: an opaque pointer of no known address space would be read by
// flat loads, which are waited for together with the LDS.
typedef const __attribute__((address_space(1))) uint8_t* GlobalBytes;

template <typename T>
__device__ __forceinline__ T global_load(GlobalBytes p, uint32_t offset) {
  return *(const __attribute__((address_space(1))) T*)(p + offset);
}

typedef __attribute__((address_space(3))) uint8_t* LdsBytes;

template <typename T>
__device__ __forceinline__ T lds_load(LdsBytes p, int offset) {
  return *(const __attribute__((address_space(3))) T*)(p + offset);
}
template <typename T>
__device__ __forceinline__ void lds_store(LdsBytes p, int offset, const T& x) {
  *(__attribute__((address_space(3))) T*)(p + offset) = x;
}

// All copies past the registers but the last kLeft are complete (any other loads under way make it
// stricter).
template <int kLeft>
__device__ __forceinline__ void wait_copies() {
  static_assert(kLeft < 64, "counted in six bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
}

// The start of a tile, opaque: added to a lane's offset it is the scalar base of the load. Seen
// through, the compiler held lane offset + head in two vector registers for each of the loads.
__device__ __forceinline__ GlobalBytes tile_base(GlobalBytes p) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+s"(p));
#endif
  return p;
}

// Byte x of four scale bytes as the scale operand of a widening conversion, which looks at bits
// 23 to 30 alone.
__device__ __forceinline__ float scale_of(uint32_t bytes, int x) {
  return __uint_as_float(__builtin_amdgcn_alignbit(bytes, bytes, 8 * x + 9));
}

// One KV head of the page arrays.
template <int D, bool kFour>
struct HeadPages {
  static constexpr int kRowBytes = kFour ? D / 2 : 2 * D, kRowScales = D / kPagedGroup;
  GlobalBytes keys, values, key_scales, value_scales;
  int page_rows, slot_mask;              // rows from one page to the next

  template <typename Args>             // with the map and the page arrays
  __device__ __forceinline__ HeadPages(const Args& a, int kvh) {
    const int64_t first = (int64_t)kvh << a.map.page_shift;
    keys = (GlobalBytes)a.key_pages + first * kRowBytes;
    values = (GlobalBytes)a.value_pages + first * kRowBytes;
    if constexpr (kFour) {
      key_scales = (GlobalBytes)a.key_scales + first * kRowScales;
      value_scales = (GlobalBytes)a.value_scales + first * kRowScales;
    }
    page_rows = a.kv_heads << a.map.page_shift;
    slot_mask = (1 << a.map.page_shift) - 1;
  }
  __device__ __forceinline__ int64_t row(int page, int p) const {
    return (int64_t)page * page_rows + (p & slot_mask);
  }
};

template <int D, bool kFour>
struct KeyTile {                         // a lane's part of 16 rows of K: row c
  u32x4 raw[D / (kFour ? 128 : 32)];
  uint32_t scale[kFour ? D / 128 : 1];   // four scale bytes of the row; the lane's is byte g

  __device__ __forceinline__ void load(const HeadPages<D, kFour>& h, int64_t row, int c, int g) {
    const GlobalBytes p = tile_base(h.keys + row * h.kRowBytes);
    if constexpr (kFour) {
      const GlobalBytes s = tile_base(h.key_scales + row * h.kRowScales);
#pragma unroll
      for (int x = 0; x < D / 128; ++x)
        raw[x] = global_load<u32x4>(p, c * (D / 2) + 64 * x + 16 * g);
      if constexpr (D == 128) {
        scale[0] = global_load<uint32_t>(s, c * 4);
      } else {
        const u32x2 w = global_load<u32x2>(s, c * 8);
        scale[0] = w[0];
        scale[1] = w[1];
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk)
        raw[kk] = global_load<u32x4>(p, c * 2 * D + 64 * kk + 16 * g);
    }
  }
  // Eight dims of the row as A operand of product kk.
  __device__ __forceinline__ u32x4 operand(int kk, int g) const {
    if constexpr (!kFour) return raw[kk];
    else return widen8(raw[kk / 4][kk % 4], scale_of(scale[kk / 4], g));
  }
  // Dim of the operand's first element.
  static __device__ __forceinline__ int dim(int kk, int g) {
    return kFour ? 128 * (kk / 4) + 32 * g + 8 * (kk % 4) : 32 * kk + 8 * g;
  }
};

}  // namespace spx
