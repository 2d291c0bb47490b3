// Paged KV cache: append with the rotary embedding applied on the way, and reading back.
//
// Append. Row (token, head) of q, k or v: the paired dims (a, b) of the first `rotary` ones
// become (a cos - b sin, b cos + a sin), cos and sin of the token's position from fp32 tables;
// v is copied. One pass: each value is read once and written once, to the page row (k, v) or
// to the caller's rotated copies (q, optionally k). Bound: HBM.
//   * A row is D / 8 lanes of 16 bytes; a lane reads its own 8 dims and, where dims are paired
//     by halves, the 8 partners (from the L1: another lane's own).
//   * bf16 rows: fp32 arithmetic, one rounding.
//   * 4-bit rows: the 32 dims of a scale are four neighbouring lanes. k is rotated in fp64
//     (bf16 x fp32 products are exact there, the sum is rounded once) and brought to fp32 by
//     rounding to odd, so that the rounding to 4 bits is that of the exact value also next to a
//     border of the grid; v needs none of it. The scale exponent is floor(log2 max) - 2, one
//     more from a mantissa of 1.75 on: the largest value is then at most one grid step off
//     (without the one more it would be clipped from 7.99 to 6).
#include "paged.h"

namespace spx {

constexpr int kPagedThreads = 256;

int paged_map(PagedMap& m, const spx_paged_cache* cache) {
  SPX_REQUIRE(cache != nullptr, SPX_EINVAL, "null cache");
  const spx_paged_cache& z = *cache;
  SPX_REQUIRE(z.head_dim == 128 || z.head_dim == 256, SPX_EUNSUPPORTED,
              "head_dim %d unsupported (128 or 256)", z.head_dim);
  SPX_REQUIRE(z.page_size >= kPagedMinPage && z.page_size <= kPagedMaxPage &&
                  (z.page_size & (z.page_size - 1)) == 0,
              SPX_EUNSUPPORTED, "page_size %d unsupported (a power of two from %d to %d)",
              z.page_size, kPagedMinPage, kPagedMaxPage);
  SPX_REQUIRE(z.batch > 0 && z.tokens > 0 && z.kv_heads > 0 && z.pages > 0 && z.table_width > 0,
              SPX_EINVAL, "bad shape: batch %d tokens %d kv_heads %d pages %d table width %d",
              z.batch, z.tokens, z.kv_heads, z.pages, z.table_width);
  SPX_REQUIRE((int64_t)z.table_width * z.page_size <= (1 << 30), SPX_EINVAL,
              "a table of %d pages of %d tokens exceeds 2^30 positions", z.table_width,
              z.page_size);
  SPX_REQUIRE(z.page_table && z.starts && z.key_pages && z.value_pages, SPX_EINVAL, "null pointer");
  SPX_REQUIRE((z.key_scales == nullptr) == (z.value_scales == nullptr), SPX_EINVAL,
              "key_scales and value_scales go together");
  auto misaligned = [](const void* x, const void* y, uintptr_t to) {
    return ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & (to - 1)) != 0;
  };
  SPX_REQUIRE(!misaligned(z.key_pages, z.value_pages, 16) &&
                  !misaligned(z.key_scales, z.value_scales, 8) &&
                  !misaligned(z.page_table, z.starts, 4) && !misaligned(z.counts, nullptr, 4),
              SPX_EINVAL,
              "pages must be 16-byte, scales 8-byte, page_table, starts and counts 4-byte aligned");
  m.table = z.page_table;
  m.table_stride = z.table_stride;
  m.starts = z.starts;
  m.counts = z.counts;
  m.width = z.table_width;
  m.pages = z.pages;
  m.page_shift = __builtin_ctz(z.page_size);
  m.kv_heads = z.kv_heads;
  return SPX_OK;
}

struct RowSource {                       // [B, T, H, D] bf16 rows
  const uint16_t* base;
  int64_t s_b, s_t, s_h;
};

struct AppendArgs {
  PagedMap map;
  RowSource q, k, v;
  const float* cos;
  const float* sin;                      // [positions, rotary / 2]; null: no rotation
  int rotary, interleaved;
  int tokens, q_heads, kv_heads, rows;   // rows: of one token, q (0 if null), k, v
  int64_t total;                         // rows of the launch
  void* key_pages;
  void* value_pages;
  uint8_t* key_scales;
  uint8_t* value_scales;
  uint16_t* q_out;                       // [B, T, Hq, D], [B, T, Hkv, D] contiguous
  uint16_t* k_out;
};

// fp64 -> fp32, rounded to odd: a later rounding to fewer bits then is that of x itself.
__device__ __forceinline__ float round_to_odd(double x) {
  const float f = (float)x;
  uint32_t u = __float_as_uint(f);
  if (__builtin_fabs((double)f) > __builtin_fabs(x)) u -= 1;    // towards zero
  if ((double)__uint_as_float(u) != x) u |= 1;
  return __uint_as_float(u);
}

__device__ __forceinline__ float fma_of(float x, float y, float z) { return __builtin_fmaf(x, y, z); }
__device__ __forceinline__ double fma_of(double x, double y, double z) {
  return __builtin_fma(x, y, z);
}

// Eight dims d0 .. d0 + 7 of a row, rotated (R = float or double).
template <typename R>
__device__ __forceinline__ void rotate8(const AppendArgs& a, const uint16_t* row, int d0, int p,
                                        const u32x4& own, R (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = (R)bf16_lo(own[e]);
    x[2 * e + 1] = (R)bf16_hi(own[e]);
  }
  if (d0 >= a.rotary) return;
  const int half = a.rotary / 2;
  if (a.interleaved) {
    const int64_t at = (int64_t)p * half + d0 / 2;
    const f32x4 c = *reinterpret_cast<const f32x4*>(a.cos + at);
    const f32x4 s = *reinterpret_cast<const f32x4*>(a.sin + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const R u = x[2 * e], w = x[2 * e + 1];
      x[2 * e] = fma_of(u, (R)c[e], -(w * (R)s[e]));
      x[2 * e + 1] = fma_of(w, (R)c[e], u * (R)s[e]);
    }
    return;
  }
  const bool low = d0 < half;
  const u32x4 other = *reinterpret_cast<const u32x4*>(row + (low ? d0 + half : d0 - half));
  const int64_t at = (int64_t)p * half + (low ? d0 : d0 - half);
  float c[8], s[8];
  load8(a.cos + at, c);
  load8(a.sin + at, s);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const R y = (R)(e & 1 ? bf16_hi(other[e / 2]) : bf16_lo(other[e / 2]));
    const R ys = y * (R)s[e];
    x[e] = fma_of(x[e], (R)c[e], low ? -ys : ys);
  }
}

// Scale byte of 32 values whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  return (uint32_t)min(max((int)((top + 0x200000u) >> 23) - 2, 2), 252);
}

__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
               pack_bf16x2(x[6], x[7])};
}

// A row of 4-bit values: the lane's 8 dims as one word, the scale by the first of the four
// lanes that share it.
template <int D>
__device__ __forceinline__ void store_4bit(void* pages, uint8_t* scales, int64_t row, int piece,
                                           const float (&x)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2));
  const uint32_t byte = scale_byte(top);
  const float scale = __uint_as_float(byte << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
  if (byte == 255) w = 0;
  if (row < 0) return;
  static_cast<uint32_t*>(pages)[row * (D / 8) + piece] = w;
  if ((piece & 3) == 0) scales[row * (D / kPagedGroup) + piece / 4] = (uint8_t)byte;
}

template <int D, bool kFour>
__global__ __launch_bounds__(kPagedThreads) void paged_append_kernel(AppendArgs a) {
  constexpr int kPieces = D / 8, kRows = kPagedThreads / kPieces;
  const int piece = threadIdx.x % kPieces, d0 = 8 * piece;
  const int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / kPieces;
  if (r >= a.total) return;
  const int64_t token = r / a.rows;
  const int in_token = (int)(r - token * a.rows);
  const int b = (int)(token / a.tokens), i = (int)(token - (int64_t)b * a.tokens);
  const int q_rows = a.rows - 2 * a.kv_heads;
  const int kind = in_token < q_rows ? 0 : in_token < q_rows + a.kv_heads ? 1 : 2;
  const int head = kind == 0 ? in_token : (in_token - q_rows) % a.kv_heads;
  const RowSource& src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
  const uint16_t* in = src.base + b * src.s_b + i * src.s_t + head * src.s_h;
  uint16_t* out = kind == 0 ? a.q_out + (token * q_rows + head) * D
                  : kind == 1 && a.k_out ? a.k_out + (token * a.kv_heads + head) * D
                                         : nullptr;
  const u32x4 own = *reinterpret_cast<const u32x4*>(in + d0);
  const int p = a.map.position(b, i);
  if (p < 0) {
    if (out) *reinterpret_cast<u32x4*>(out + d0) = u32x4{};
    return;
  }
  const int page = kind == 0 ? -1 : a.map.page(b, p);
  const int64_t row = page < 0 ? -1 : a.map.row(page, head, p);
  void* pages = kind == 1 ? a.key_pages : a.value_pages;
  const bool turn = kind < 2 && a.cos != nullptr;
  float x[8];
  if (kFour && kind == 1 && turn) {
    double y[8];
    rotate8<double>(a, in, d0, p, own, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = round_to_odd(y[e]);
    if (out) *reinterpret_cast<u32x4*>(out + d0) = pack8(x);
    store_4bit<D>(pages, a.key_scales, row, piece, x);
    return;
  }
  u32x4 packed = own;
  if (turn) {
    rotate8<float>(a, in, d0, p, own, x);
    packed = pack8(x);
  }
  if (out) *reinterpret_cast<u32x4*>(out + d0) = packed;
  if (kind == 0) return;
  if (kFour) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = bf16_lo(own[e]);
      x[2 * e + 1] = bf16_hi(own[e]);
    }
    store_4bit<D>(pages, kind == 1 ? a.key_scales : a.value_scales, row, piece, x);
  } else if (row >= 0) {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(pages) + row * D + d0) = packed;
  }
}

struct GatherArgs {
  PagedMap map;
  const void* key_pages;
  const void* value_pages;
  const uint8_t* key_scales;
  const uint8_t* value_scales;
  int tokens, kv_heads;
  int64_t total;                         // rows of the launch, k then v of each token
  uint16_t* k_out;                       // [B, T, Hkv, D] contiguous
  uint16_t* v_out;
};

template <int D, bool kFour>
__global__ __launch_bounds__(kPagedThreads) void paged_gather_kernel(GatherArgs a) {
  constexpr int kPieces = D / 8, kRows = kPagedThreads / kPieces;
  const int piece = threadIdx.x % kPieces;
  const int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / kPieces;
  if (r >= a.total) return;
  const int64_t token = r / (2 * a.kv_heads);
  const int in_token = (int)(r - token * 2 * a.kv_heads);
  const int b = (int)(token / a.tokens), i = (int)(token - (int64_t)b * a.tokens);
  const bool is_v = in_token >= a.kv_heads;
  const int head = is_v ? in_token - a.kv_heads : in_token;
  const int p = a.map.position(b, i);
  const int page = p < 0 ? -1 : a.map.page(b, p);
  u32x4 x{};
  if (page >= 0) {
    const int64_t row = a.map.row(page, head, p);
    const void* pages = is_v ? a.value_pages : a.key_pages;
    if (kFour) {
      const uint8_t* scales = is_v ? a.value_scales : a.key_scales;
      const uint32_t byte = scales[row * (D / kPagedGroup) + piece / 4];
      x = widen8(static_cast<const uint32_t*>(pages)[row * kPieces + piece],
                 __uint_as_float(byte << 23));
    } else {
      x = static_cast<const u32x4*>(pages)[row * kPieces + piece];
    }
  }
  uint16_t* out = is_v ? a.v_out : a.k_out;
  reinterpret_cast<u32x4*>(out)[(token * a.kv_heads + head) * kPieces + piece] = x;
}

static int row_source(RowSource& r, const void* base, const int64_t* strides, const char* name) {
  SPX_REQUIRE(base && strides, SPX_EINVAL, "null pointer (%s)", name);
  SPX_REQUIRE((reinterpret_cast<uintptr_t>(base) & 15) == 0 && strides[3] == 1 &&
                  ((strides[0] | strides[1] | strides[2]) & 7) == 0,
              SPX_EINVAL,
              "%s: base must be 16-byte aligned, the dim stride 1, the others multiples of 8", name);
  r.base = static_cast<const uint16_t*>(base);
  r.s_b = strides[0];
  r.s_t = strides[1];
  r.s_h = strides[2];
  return SPX_OK;
}

template <int D>
static unsigned row_blocks(int64_t rows) {
  constexpr int kRows = kPagedThreads / (D / 8);
  return (unsigned)((rows + kRows - 1) / kRows);
}

}  // namespace spx

using namespace spx;

extern "C" int spx_paged_append(const spx_paged_cache* cache, const void* q,
                                const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                const void* v, const int64_t* v_strides, int q_heads,
                                const float* rope_cos, const float* rope_sin, int rope_positions,
                                int rotary_dim, int interleaved, void* q_out, void* k_out,
                                void* stream) {
  AppendArgs a{};
  int status = paged_map(a.map, cache);
  if (status != SPX_OK) return status;
  SPX_REQUIRE(q == nullptr || (q_heads > 0 && q_out), SPX_EINVAL, "q needs q_heads and q_out");
  if (q != nullptr && (status = row_source(a.q, q, q_strides, "q")) != SPX_OK) return status;
  if ((status = row_source(a.k, k, k_strides, "k")) != SPX_OK) return status;
  if ((status = row_source(a.v, v, v_strides, "v")) != SPX_OK) return status;
  SPX_REQUIRE((rope_cos == nullptr) == (rope_sin == nullptr), SPX_EINVAL,
              "rope_cos and rope_sin go together");
  if (rope_cos != nullptr) {
    SPX_REQUIRE(rotary_dim > 0 && rotary_dim <= cache->head_dim && rotary_dim % 16 == 0,
                SPX_EUNSUPPORTED, "rotary_dim %d unsupported (a multiple of 16 up to head_dim %d)",
                rotary_dim, cache->head_dim);
    SPX_REQUIRE(rope_positions >= (int64_t)cache->table_width * cache->page_size, SPX_EINVAL,
                "the rope table has %d positions, the page table reaches %lld", rope_positions,
                (long long)cache->table_width * cache->page_size);
    SPX_REQUIRE(((reinterpret_cast<uintptr_t>(rope_cos) | reinterpret_cast<uintptr_t>(rope_sin)) &
                 15) == 0, SPX_EINVAL, "rope tables must be 16-byte aligned");
  }
  SPX_REQUIRE(((reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_out)) & 15) == 0,
              SPX_EINVAL, "outputs must be 16-byte aligned");
  a.cos = rope_cos; a.sin = rope_sin;
  a.rotary = rope_cos ? rotary_dim : 0;
  a.interleaved = interleaved;
  a.tokens = cache->tokens;
  a.kv_heads = cache->kv_heads;
  const int64_t rows = (q ? q_heads : 0) + 2 * (int64_t)a.kv_heads;
  SPX_REQUIRE(rows <= 0x7fffffff && (double)cache->batch * cache->tokens * rows <= 0x1p33,
              SPX_EINVAL, "more than 2^33 rows in a call");
  a.rows = (int)rows;
  a.total = (int64_t)cache->batch * cache->tokens * rows;
  a.key_pages = cache->key_pages; a.value_pages = cache->value_pages;
  a.key_scales = static_cast<uint8_t*>(cache->key_scales);
  a.value_scales = static_cast<uint8_t*>(cache->value_scales);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_out = static_cast<uint16_t*>(k_out);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool four = cache->key_scales != nullptr;
  if (cache->head_dim == 128) {
    const unsigned blocks = row_blocks<128>(a.total);
    if (four) paged_append_kernel<128, true><<<blocks, kPagedThreads, 0, st>>>(a);
    else paged_append_kernel<128, false><<<blocks, kPagedThreads, 0, st>>>(a);
  } else {
    const unsigned blocks = row_blocks<256>(a.total);
    if (four) paged_append_kernel<256, true><<<blocks, kPagedThreads, 0, st>>>(a);
    else paged_append_kernel<256, false><<<blocks, kPagedThreads, 0, st>>>(a);
  }
  return launch_status("paged_append");
}

extern "C" int spx_paged_gather(const spx_paged_cache* cache, void* k_out, void* v_out,
                                void* stream) {
  GatherArgs a{};
  const int status = paged_map(a.map, cache);
  if (status != SPX_OK) return status;
  SPX_REQUIRE(k_out && v_out &&
                  ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) ==
                      0,
              SPX_EINVAL, "outputs null or not 16-byte aligned");
  a.key_pages = cache->key_pages; a.value_pages = cache->value_pages;
  a.key_scales = static_cast<const uint8_t*>(cache->key_scales);
  a.value_scales = static_cast<const uint8_t*>(cache->value_scales);
  a.tokens = cache->tokens;
  a.kv_heads = cache->kv_heads;
  SPX_REQUIRE(2.0 * cache->batch * cache->tokens * cache->kv_heads <= 0x1p33 &&
                  cache->kv_heads <= 1 << 29,
              SPX_EINVAL, "more than 2^33 rows in a call");
  a.total = (int64_t)cache->batch * cache->tokens * 2 * cache->kv_heads;
  a.k_out = static_cast<uint16_t*>(k_out);
  a.v_out = static_cast<uint16_t*>(v_out);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool four = cache->key_scales != nullptr;
  if (cache->head_dim == 128) {
    const unsigned blocks = row_blocks<128>(a.total);
    if (four) paged_gather_kernel<128, true><<<blocks, kPagedThreads, 0, st>>>(a);
    else paged_gather_kernel<128, false><<<blocks, kPagedThreads, 0, st>>>(a);
  } else {
    const unsigned blocks = row_blocks<256>(a.total);
    if (four) paged_gather_kernel<256, true><<<blocks, kPagedThreads, 0, st>>>(a);
    else paged_gather_kernel<256, false><<<blocks, kPagedThreads, 0, st>>>(a);
  }
  return launch_status("paged_gather");
}
