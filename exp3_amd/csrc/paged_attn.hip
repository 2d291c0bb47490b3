// Attention of new tokens over a paged KV cache (bf16 or 4-bit pages, fp32 softmax and
// accumulation): one workgroup per (sequence, token, query head), one key per wave and step.
#include "paged.h"

namespace spx {

constexpr int kPaThreads = 256, kPaWaves = kPaThreads / 64;

struct PagedAttnArgs {
  PagedMap map;
  const uint16_t* q;
  int64_t qs_b, qs_t, qs_h;
  const void* key_pages;
  const void* value_pages;
  const uint8_t* key_scales;
  const uint8_t* value_scales;
  int tokens, q_heads, kv_heads, group;
  float scale_log2;
  uint16_t* out;
  float* lse;
};

// dims (D / 64) lane .. of a row, as fp32
template <int D, bool kFour>
__device__ __forceinline__ void load_row(const void* pages, const uint8_t* scales, int64_t row,
                                         int lane, float (&x)[D / 64]) {
  constexpr int N = D / 64;
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    const int64_t at = row * (D / 2) + (lane * N + e) / 2;       // pairs of dims
    uint32_t w;
    if (kFour) {
      const uint32_t byte = scales[row * (D / kPagedGroup) + lane * N / kPagedGroup];
      w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(
                                           (uint32_t) static_cast<const uint8_t*>(pages)[at],
                                           __uint_as_float(byte << 23), 0));
    } else {
      w = static_cast<const uint32_t*>(pages)[at];
    }
    x[e] = bf16_lo(w);
    x[e + 1] = bf16_hi(w);
  }
}

template <int D, bool kFour>
__global__ __launch_bounds__(kPaThreads) void paged_attn_kernel(PagedAttnArgs a) {
  constexpr int N = D / 64;
  __shared__ float part_m[kPaWaves], part_l[kPaWaves], part_o[kPaWaves][D];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t out_row = blockIdx.x;
  const int h = (int)(out_row % a.q_heads), i = (int)(out_row / a.q_heads % a.tokens);
  const int b = (int)(out_row / a.q_heads / a.tokens), kvh = h / a.group;
  const int last = a.map.position(b, i);
  const uint16_t* qr = a.q + b * a.qs_b + i * a.qs_t + h * a.qs_h + lane * N;
  float q[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    q[e] = __uint_as_float((uint32_t)qr[e] << 16);
    o[e] = 0.0f;
  }
  for (int p = w; p <= last; p += kPaWaves) {
    const int page = a.map.page(b, p);
    if (page < 0) continue;
    const int64_t row = a.map.row(page, kvh, p);
    float k[N], v[N];
    load_row<D, kFour>(a.key_pages, a.key_scales, row, lane, k);
    load_row<D, kFour>(a.value_pages, a.value_scales, row, lane, v);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) s += q[e] * k[e];
    s = wave_sum(s) * a.scale_log2;
    const float m_new = max_nan(m, s);
    const float shift = m_new == -INFINITY ? 0.0f : m_new;
    const float corr = exp2_fast(m - shift), prob = exp2_fast(s - shift);
    l = l * corr + prob;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = o[e] * corr + prob * v[e];
    m = m_new;
  }
  if (lane == 0) {
    part_m[w] = m;
    part_l[w] = l;
  }
#pragma unroll
  for (int e = 0; e < N; ++e) part_o[w][lane * N + e] = o[e];
  block_sync();
  float top = part_m[0], sum = 0.0f;
#pragma unroll
  for (int x = 1; x < kPaWaves; ++x) top = max_nan(top, part_m[x]);
  const float shift = top == -INFINITY ? 0.0f : top;
  float wt[kPaWaves];
#pragma unroll
  for (int x = 0; x < kPaWaves; ++x) {
    wt[x] = exp2_fast(part_m[x] - shift);
    sum += wt[x] * part_l[x];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int d = threadIdx.x; d < D; d += kPaThreads) {
    float acc = 0.0f;
#pragma unroll
    for (int x = 0; x < kPaWaves; ++x) acc += wt[x] * part_o[x][d];
    a.out[out_row * D + d] = to_bf16_bits(acc * inv);
  }
  if (threadIdx.x == 0 && a.lse)
    a.lse[out_row] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

}  // namespace spx

using namespace spx;

extern "C" int64_t spx_paged_attention_workspace_bytes(int table_width, int page_size, int max_keys,
                                                       int batch, int tokens, int q_heads,
                                                       int kv_heads, int head_dim) {
  if (table_width <= 0 || page_size <= 0 || max_keys < 0 || batch <= 0 || tokens <= 0 ||
      q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || (head_dim != 128 && head_dim != 256))
    return -1;
  return 0;
}

extern "C" int spx_paged_attention(const void* q, const int64_t* q_strides,
                                   const int32_t* page_table, int64_t table_stride, int table_width,
                                   const int32_t* starts, const int32_t* counts,
                                   const void* key_pages, const void* value_pages,
                                   const void* key_scales, const void* value_scales, int pages,
                                   int page_size, int max_keys, int batch, int tokens, int q_heads,
                                   int kv_heads, int head_dim, float scale, void* workspace,
                                   void* out, float* lse, void* stream) {
  PagedAttnArgs a{};
  const int status = paged_map(a.map, page_table, table_stride, table_width, starts, counts,
                               key_pages, value_pages, key_scales, value_scales, pages, page_size,
                               batch, tokens, kv_heads, head_dim);
  if (status != SPX_OK) return status;
  SPX_REQUIRE(q_heads > 0 && q_heads % kv_heads == 0 && max_keys >= 0, SPX_EINVAL,
              "bad shape: q_heads %d kv_heads %d max_keys %d", q_heads, kv_heads, max_keys);
  SPX_REQUIRE(q && q_strides && out, SPX_EINVAL, "null pointer");
  SPX_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 &&
                  q_strides[3] == 1 && ((q_strides[0] | q_strides[1] | q_strides[2]) & 7) == 0,
              SPX_EINVAL,
              "q, out: bases must be 16-byte aligned, q's dim stride 1, the others multiples of 8");
  const int64_t rows = (int64_t)batch * tokens * q_heads;
  SPX_REQUIRE(rows <= 0x7fffffff, SPX_EINVAL, "more than 2^31 - 1 query rows");
  a.q = static_cast<const uint16_t*>(q);
  a.qs_b = q_strides[0]; a.qs_t = q_strides[1]; a.qs_h = q_strides[2];
  a.key_pages = key_pages; a.value_pages = value_pages;
  a.key_scales = static_cast<const uint8_t*>(key_scales);
  a.value_scales = static_cast<const uint8_t*>(value_scales);
  a.tokens = tokens; a.q_heads = q_heads; a.kv_heads = kv_heads; a.group = q_heads / kv_heads;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (head_dim == 128) {
    if (key_scales) paged_attn_kernel<128, true><<<(unsigned)rows, kPaThreads, 0, st>>>(a);
    else paged_attn_kernel<128, false><<<(unsigned)rows, kPaThreads, 0, st>>>(a);
  } else {
    if (key_scales) paged_attn_kernel<256, true><<<(unsigned)rows, kPaThreads, 0, st>>>(a);
    else paged_attn_kernel<256, false><<<(unsigned)rows, kPaThreads, 0, st>>>(a);
  }
  return launch_status("paged_attention");
}
