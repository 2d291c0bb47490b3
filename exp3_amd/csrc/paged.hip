// Paged KV cache: append with the rotary embedding applied on the way, and reading back.
//
// Append. Row (token, head) of q, k or v: the paired dims (a, b) of the first `rotary` ones
// become (a cos - b sin, b cos + a sin), cos and sin of the token's position from fp32 tables;
// v is copied. One pass: each value is read once and written once, to the page row (k, v) or
// to the caller's rotated copies (q, optionally k). Bound: HBM: 32640 tokens (28/4 heads, bf16, with
// both copies) 110 us for 652 MB, 5.9 TB/s where a large elementwise kernel reaches 6.2.
//   * A row is D / 8 lanes of 16 bytes, 8 dims each; where dims are paired by halves the partners
//     come from the lane that holds them.
//   * bf16 rows: fp32 arithmetic, one rounding.
//   * 4-bit rows: the 32 dims of a scale are four neighbouring lanes. k is rotated in fp64
//     (bf16 x fp32 products are exact there, the sum is rounded once) and brought to fp32 by
//     rounding to odd, so that the rounding to 4 bits is that of the exact value also next to a
//     border of the grid; v needs none of it. The scale exponent is floor(log2 max) - 2, one
//     more from a mantissa of 1.75 on: the largest value is then at most one grid step off
//     (without the one more it would be clipped from 7.99 to 6).
#include <algorithm>

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
  SPX_REQUIRE(z.kv_heads <= 1 << 16, SPX_EINVAL, "%d KV heads are more than 2^16", z.kv_heads);
  SPX_REQUIRE(z.batch <= 1 << 30, SPX_EINVAL, "%d sequences are more than 2^30", z.batch);
  SPX_REQUIRE(z.reserved == 0, SPX_EINVAL, "reserved must be 0");
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
  int batch, tokens, q_rows, kv_heads;   // q_rows: query heads, 0 without q
  int wave_shift;                        // 2^wave_shift waves share a token's rows
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

// Calls of 8 MB and more store their outputs past the caches. The size is that of all rows in bf16,
// read and written, also where pages of 4 bits make it less. Through the caches and past them, us (28/4
// heads, six calls in turn; the first figure into memory that the calls hand on to each other, the
// second into memory of each call's own):
//              append, bf16           append, 4 bits         gather, bf16           gather, 4 bits
//     4 MB   5.2  5.2 ->  5.1  5.1  5.2  5.2 ->  5.1  5.0  3.9  3.7 ->  3.4  3.5  3.8  3.7 ->  3.8  3.6
//     8 MB   5.6  5.5 ->  5.4  5.4  5.5  5.4 ->  5.4  5.3  4.4  4.4 ->  4.3  4.3  4.1  4.1 ->  4.0  4.0
//    16 MB   6.8  6.8 ->  6.3  6.3  6.8  6.8 ->  6.4  6.4  5.6  5.6 ->  5.4  5.4  5.0  4.9 ->  4.4  4.4
//    64 MB  16.2 18.0 -> 16.3 16.2 15.9 17.1 -> 13.8 13.6 12.4 16.3 -> 12.3 12.3 10.1 10.6 ->  9.3  9.4
//   128 MB  26.8 30.3 -> 29.0 28.8 27.8 30.8 -> 30.3 30.1 25.0 28.0 -> 26.4 26.3 16.1 22.7 -> 15.8 15.4
// Below 4 MB both are equal. A dense prefill behind the append takes as long in all (16000 tokens 1632
// and 1632 us, 1089 43.6 and 42.8). What a decode step writes is read at once and stays: attention
// behind it 36.3 us with it in the cache, 37.1 past it.
constexpr int64_t kStreamedBytes = 8 << 20;

// (A template parameter: of a run-time choice the compiler makes one ordinary store.)
template <bool kStreamed>
__device__ __forceinline__ void store_row(uint16_t* p, const u32x4& x) {
  if constexpr (kStreamed) __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(p));
  else *reinterpret_cast<u32x4*>(p) = x;
}

__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
               pack_bf16x2(x[6], x[7])};
}

// A lane's part of the rotation of a token: its eight dims 8 piece .. 8 piece + 7.
struct Rotation {
  bool turns, interleaved;
  float c[8], s[8];

  // First of the dims that these are paired with (themselves if they are paired inside or not).
  static __device__ __forceinline__ int partner(const AppendArgs& a, int d0) {
    const int half = a.rotary / 2;
    return d0 >= a.rotary || a.interleaved ? d0 : d0 < half ? d0 + half : d0 - half;
  }

  __device__ __forceinline__ Rotation(const AppendArgs& a, int d0, int p) {
    turns = a.cos != nullptr && d0 < a.rotary;
    interleaved = a.interleaved != 0;
    if (!turns) return;
    const int half = a.rotary / 2;
    const bool low = d0 < half;
    if (interleaved) {
      const int64_t at = (int64_t)p * half + d0 / 2;
      const f32x4 x = *reinterpret_cast<const f32x4*>(a.cos + at);
      const f32x4 y = *reinterpret_cast<const f32x4*>(a.sin + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[2 * e] = c[2 * e + 1] = x[e];
        s[2 * e] = -y[e];
        s[2 * e + 1] = y[e];
      }
    } else {
      const int64_t at = (int64_t)p * half + (low ? d0 : d0 - half);
      load8(a.cos + at, c);
      load8(a.sin + at, s);
      if (low)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = -s[e];
    }
  }
  // Dim e; R = float or double; `other`: the partner dims (or the same ones).
  template <typename R>
  __device__ __forceinline__ R dim(const u32x4& own, const u32x4& other, int e) const {
    const R mine = (R)(e & 1 ? bf16_hi(own[e / 2]) : bf16_lo(own[e / 2]));
    const uint32_t w = interleaved ? own[e / 2] : other[e / 2];
    const bool high = interleaved ? !(e & 1) : e & 1;
    const R paired = (R)(high ? bf16_hi(w) : bf16_lo(w));
    return fma_of(mine, (R)c[e], paired * (R)s[e]);
  }
  __device__ __forceinline__ u32x4 rotated(const u32x4& own, const u32x4& other) const {
    if (!turns) return own;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = dim<float>(own, other, e);
    return pack8(x);
  }
};

// Waits for a load's result.
__device__ __forceinline__ void arrived(u32x4& x) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(x));
#endif
}

// Scale byte of 32 values whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  return (uint32_t)min(max((int)((top + 0x200000u) >> 23) - 2, 2), 252);
}

__device__ __forceinline__ void unpack8(const u32x4& w, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = bf16_lo(w[e]);
    x[2 * e + 1] = bf16_hi(w[e]);
  }
}

// A row of 4-bit values: the lane's 8 dims as one word, the scale by all four lanes that
// share it.
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
  static_cast<uint32_t*>(pages)[row * (D / 8) + piece] = w;
  scales[row * (D / kPagedGroup) + piece / 4] = (uint8_t)byte;
}

// A token is one wave's, or several waves' that share its chunks. A chunk is kRows heads of v, k or
// q, so what is done with it is uniform in the wave; lanes behind the last head repeat it (and store
// the same again). The next chunk is loaded while one is rotated, and every chunk of q is one load and
// one store: the wait for the load then counts past the store behind it. (A row per group of lanes of
// any kind, stores under conditions, waited for each store as well: 32640 tokens, 28/4 heads, bf16,
// rotated copies of q and k, 142 -> 120 us; 8000 tokens 48 -> 29, 4 x up to 2113 in 4 bits 62 -> 35.) What a token's
// chunks have in common (its place, cos and sin of the lane's dims) is found once, behind the first
// load. Two chunks ahead: no change.
template <int D, bool kFour, bool kStreamed>
__global__ __launch_bounds__(kPagedThreads, kFour ? 6 : 1) void paged_append_kernel(AppendArgs a) {
  constexpr int kPieces = D / 8, kRows = kWave / kPieces;        // lanes of a row, heads of a chunk
  const int lane = threadIdx.x & 63, piece = lane % kPieces, d0 = 8 * piece;
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kPagedThreads / kWave) +
                                                  threadIdx.x / kWave);
  const int i = wave >> a.wave_shift, part = wave & ((1 << a.wave_shift) - 1);
  if (i >= a.tokens) return;
  const int q_chunks = (a.q_rows + kRows - 1) / kRows, kv_chunks = (a.kv_heads + kRows - 1) / kRows;
  const int chunks = q_chunks + 2 * kv_chunks, step = 1 << a.wave_shift;
  const int sub = lane / kPieces;
  const int from = lane - piece + Rotation::partner(a, d0) / 8;  // the lane of the paired dims
  const unsigned b = blockIdx.z * gridDim.y + blockIdx.y;
  if (b >= (unsigned)a.batch || part >= chunks) return;
  const auto head_of = [&](int chunk, int heads) { return min(chunk * kRows + sub, heads - 1); };
  const auto load = [&](int n) {       // chunks of v, of k, of q
    const bool is_v = n < kv_chunks, is_k = !is_v && n < 2 * kv_chunks;
    const RowSource& src = is_v ? a.v : is_k ? a.k : a.q;
    const int chunk = n - (is_v ? 0 : is_k ? kv_chunks : 2 * kv_chunks);
    const uint16_t* in = src.base + b * src.s_b + i * src.s_t;
    return *reinterpret_cast<const u32x4*>(
        in + head_of(chunk, is_v || is_k ? a.kv_heads : a.q_rows) * src.s_h + d0);
  };
  const auto partners = [&](const u32x4& own) {
    u32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (uint32_t)__shfl((int)own[e], from);
    return x;
  };
  int n = part;
  u32x4 next = load(n);
  const auto advance = [&] {
    const u32x4 own = next;
    n += step;
    next = load(min(n, chunks - 1));
    return own;
  };
  const int p = a.map.position(b, i), page = a.map.uniform_page(b, p);
  const int64_t token = (int64_t)b * a.tokens + i;
  uint16_t* const q_out = a.q_out + token * a.q_rows * D + d0;
  uint16_t* const k_out = a.k_out ? a.k_out + token * a.kv_heads * D + d0 : nullptr;
  if (p < 0) {
    for (; n < chunks; n += step) {
      if (n >= 2 * kv_chunks)
        store_row<kStreamed>(q_out + head_of(n - 2 * kv_chunks, a.q_rows) * D, u32x4{});
      else if (n >= kv_chunks && k_out)
        store_row<kStreamed>(k_out + head_of(n - kv_chunks, a.kv_heads) * D, u32x4{});
    }
    return;
  }
  const Rotation rotation(a, d0, p);
  while (n < kv_chunks) {
    const int64_t row = a.map.row(page, head_of(n, a.kv_heads), p);
    const u32x4 own = advance();
    if (page < 0) continue;
    if constexpr (kFour) {
      float x[8];
      unpack8(own, x);
      store_4bit<D>(a.value_pages, a.value_scales, row, piece, x);
    } else {
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.value_pages) + row * D + d0) = own;
    }
  }
  while (n < 2 * kv_chunks) {
    const int head = head_of(n - kv_chunks, a.kv_heads);
    const int64_t row = a.map.row(page, head, p);
    const u32x4 own = advance(), other = partners(own);
    u32x4 packed = own;
    if constexpr (kFour) {
      float x[8];
      if (rotation.turns) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = round_to_odd(rotation.dim<double>(own, other, e));
          if (e % 2) __builtin_amdgcn_sched_barrier(0);        // two at a time: registers
        }
        packed = pack8(x);
      } else {
        unpack8(own, x);
      }
      if (page >= 0) store_4bit<D>(a.key_pages, a.key_scales, row, piece, x);
    } else {
      packed = rotation.rotated(own, other);
      if (page >= 0)
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.key_pages) + row * D + d0) = packed;
    }
    if (k_out) store_row<kStreamed>(k_out + head * D, packed);
  }
  // Here first, so that the loop's wait for a load is not one for the store behind it.
  arrived(next);
  const uint16_t* q_in = a.q.base + b * a.q.s_b + i * a.q.s_t + d0;
  for (int chunk = n - 2 * kv_chunks; chunk < q_chunks; chunk += step) {
    const u32x4 own = next;
    next = *reinterpret_cast<const u32x4*>(
        q_in + head_of(min(chunk + step, q_chunks - 1), a.q_rows) * a.q.s_h);
    const u32x4 other = partners(own);
    const u32x4 packed = rotation.rotated(own, other);
    store_row<kStreamed>(q_out + head_of(chunk, a.q_rows) * D, packed);
  }
}

struct GatherArgs {
  PagedMap map;
  const void* key_pages;
  const void* value_pages;
  const uint8_t* key_scales;
  const uint8_t* value_scales;
  int batch, tokens, kv_heads, wave_shift;
  uint16_t* k_out;                       // [B, T, Hkv, D] contiguous
  uint16_t* v_out;
};

// A lane's dims of a stored row.
template <int D, bool kFour>
struct StoredPart {
  u32x4 raw;
  uint32_t byte;
  // Row r of a token: keys, then values.
  __device__ __forceinline__ void load(const GatherArgs& a, int page, int p, int r, int piece) {
    if (r >= 2 * a.kv_heads || page < 0) return;
    const bool is_v = r >= a.kv_heads;
    const int64_t row = a.map.row(page, is_v ? r - a.kv_heads : r, p);
    const void* pages = is_v ? a.value_pages : a.key_pages;
    if constexpr (kFour) {
      raw[0] = static_cast<const uint32_t*>(pages)[row * (D / 8) + piece];
      byte = (is_v ? a.value_scales : a.key_scales)[row * (D / kPagedGroup) + piece / 4];
    } else {
      raw = static_cast<const u32x4*>(pages)[row * (D / 8) + piece];
    }
  }
  __device__ __forceinline__ u32x4 value() const {
    if constexpr (kFour) return widen8(raw[0], __uint_as_float(byte << 23));
    else return raw;
  }
};

// Waves and tokens as in the append kernel.
template <int D, bool kFour, bool kStreamed>
__global__ __launch_bounds__(kPagedThreads) void paged_gather_kernel(GatherArgs a) {
  constexpr int kPieces = D / 8, kRows = kWave / kPieces;
  const int lane = threadIdx.x & 63, piece = lane % kPieces;
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kPagedThreads / kWave) +
                                                  threadIdx.x / kWave);
  const int i = wave >> a.wave_shift, part = wave & ((1 << a.wave_shift) - 1);
  if (i >= a.tokens) return;
  const int rows = 2 * a.kv_heads, step = kRows << a.wave_shift;
  const int first = part * kRows + lane / kPieces;
  const unsigned b = blockIdx.z * gridDim.y + blockIdx.y;
  if (b >= (unsigned)a.batch) return;
  const int p = a.map.position(b, i), page = a.map.uniform_page(b, p);
  const int64_t token = (int64_t)b * a.tokens + i;
  StoredPart<D, kFour> next;
  next.load(a, page, p, first, piece);
  for (int r = first; r < rows; r += step) {
    const StoredPart<D, kFour> now = next;
    next.load(a, page, p, r + step, piece);
    const bool is_v = r >= a.kv_heads;
    uint16_t* out = is_v ? a.v_out : a.k_out;
    const int64_t row = token * a.kv_heads + (is_v ? r - a.kv_heads : r);
    store_row<kStreamed>(out + row * D + 8 * piece, page < 0 ? u32x4{} : now.value());
  }
}

// Waves of a token: as many as it has chunks while the launch has fewer than 2048. With bf16 pages
// also while a wave keeps more than two chunks and there are fewer than 65536: 8000 tokens 31 -> 29 us,
// 32640 126 -> 119; 4-bit pages 35 -> 36 us, 16000 tokens 63 -> 70 (the rotation of k at one end).
static int token_waves(int64_t tokens, int64_t rows, int head_dim, bool four) {
  const int wave_rows = kWave / (head_dim / 8);
  int shift = 0;
  while (tokens << shift < 2048 && (int64_t)wave_rows << shift < rows) ++shift;
  while (!four && tokens << shift < 65536 && (int64_t)wave_rows << shift < rows / 4) ++shift;
  return shift;
}

static dim3 token_grid(int batch, int tokens, int wave_shift) {
  const int waves = kPagedThreads / kWave;
  return dim3((unsigned)((((int64_t)tokens << wave_shift) + waves - 1) / waves),
              (unsigned)std::min(batch, 65535), (unsigned)((batch + 65534) / 65535));
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
static void launch_append(const AppendArgs& a, bool four, bool streamed, dim3 grid, hipStream_t st) {
  if (four && streamed) paged_append_kernel<D, true, true><<<grid, kPagedThreads, 0, st>>>(a);
  else if (four) paged_append_kernel<D, true, false><<<grid, kPagedThreads, 0, st>>>(a);
  else if (streamed) paged_append_kernel<D, false, true><<<grid, kPagedThreads, 0, st>>>(a);
  else paged_append_kernel<D, false, false><<<grid, kPagedThreads, 0, st>>>(a);
}

template <int D>
static void launch_gather(const GatherArgs& a, bool four, bool streamed, dim3 grid, hipStream_t st) {
  if (four && streamed) paged_gather_kernel<D, true, true><<<grid, kPagedThreads, 0, st>>>(a);
  else if (four) paged_gather_kernel<D, true, false><<<grid, kPagedThreads, 0, st>>>(a);
  else if (streamed) paged_gather_kernel<D, false, true><<<grid, kPagedThreads, 0, st>>>(a);
  else paged_gather_kernel<D, false, false><<<grid, kPagedThreads, 0, st>>>(a);
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
  a.batch = cache->batch;
  a.tokens = cache->tokens;
  a.kv_heads = cache->kv_heads;
  a.q_rows = q ? q_heads : 0;
  const int64_t rows = a.q_rows + 2 * (int64_t)a.kv_heads;
  SPX_REQUIRE(rows <= 1 << 20 && cache->tokens <= 1 << 24, SPX_EINVAL,
              "more than 2^20 heads or 2^24 tokens in a call");
  const bool four = cache->key_scales != nullptr;
  a.wave_shift = token_waves((int64_t)a.batch * a.tokens, rows, cache->head_dim, four);
  const bool streamed =
      (int64_t)a.batch * a.tokens * rows * cache->head_dim * 4 >= kStreamedBytes;
  a.key_pages = cache->key_pages; a.value_pages = cache->value_pages;
  a.key_scales = static_cast<uint8_t*>(cache->key_scales);
  a.value_scales = static_cast<uint8_t*>(cache->value_scales);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_out = static_cast<uint16_t*>(k_out);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid = token_grid(a.batch, a.tokens, a.wave_shift);
  if (cache->head_dim == 128) launch_append<128>(a, four, streamed, grid, st);
  else launch_append<256>(a, four, streamed, grid, st);
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
  a.batch = cache->batch;
  a.tokens = cache->tokens;
  a.kv_heads = cache->kv_heads;
  SPX_REQUIRE(a.tokens <= 1 << 24, SPX_EINVAL, "more than 2^24 tokens in a call");
  const bool four = cache->key_scales != nullptr;
  a.wave_shift = token_waves((int64_t)a.batch * a.tokens, 2 * a.kv_heads, cache->head_dim, four);
  const bool streamed =
      (int64_t)a.batch * a.tokens * 2 * a.kv_heads * cache->head_dim * 4 >= kStreamedBytes;
  a.k_out = static_cast<uint16_t*>(k_out);
  a.v_out = static_cast<uint16_t*>(v_out);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid = token_grid(a.batch, a.tokens, a.wave_shift);
  if (cache->head_dim == 128) launch_gather<128>(a, four, streamed, grid, st);
  else launch_gather<256>(a, four, streamed, grid, st);
  return launch_status("paged_gather");
}
