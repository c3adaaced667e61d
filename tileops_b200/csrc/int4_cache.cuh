// Layout and arithmetic of the 4-bit paged KV cache, shared by its writer (qk_norm_rope.cu), its reader for a
// prefill (int4_cache.cu) and the decode attention (gqa_decode_int4.cu).
//
// kv_pages is uint8 [pages, heads_kv, page_size * (dim + 8)].  The bytes of one (page, KV head) are page_size / 16
// RECORDS of 16 tokens:
//     K codes  [16][dim / 2]     dim 2j of a token in the low half of byte j, dim 2j + 1 in the high half
//     V codes  [16][dim / 2]
//     params   [16][4] float16   K scale, K offset, V scale, V offset
// and value = scale * code + offset.  A record is contiguous, so whatever the page size is a tile of the attention is
// a few untiled bulk copies of whole records (2176 bytes at head dim 128, 1152 at 64), K, V and parameters together.
//
// Quantiser of one row (one token of one KV head), 15 steps between its smallest and largest value:
//     lo, hi = min, max of the values clamped to +-65504
//     even slots: offset = f16(lo), scale =  f16((hi - lo) / 15)
//     odd slots:  offset = f16(hi), scale = -f16((hi - lo) / 15)
//     code = clamp(rint((x - offset) * (1 / scale)), 0, 15), 0 where scale == 0
// in fp32 with one reciprocal per row.  Both signs decode the same way.  They alternate because the attention sums
// p * scale * code over thousands of tokens in tensor-core accumulators: codes are 0..15, so sums of one sign would
// grow with the context while their useful part, the deviations from the mean, grows with its square root, and the
// accumulator's rounding would eat into it; with alternating signs the means cancel.
// A row that holds a NaN gets NaN parameters: its values, and the outputs that attend to it, are NaN.
#pragma once

#include <type_traits>

#include "tb200_common.cuh"

namespace tb200 {

constexpr int kInt4Tokens = 16;   // tokens of a record
__host__ __device__ constexpr int int4_record_bytes(int dim) { return kInt4Tokens * (dim + 8); }
constexpr float kInt4Clamp = 65504.f;   // largest float16

// min and max that pass a NaN on
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// the same of two 16-bit values side by side
template <typename T>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t y;
  if constexpr (std::is_same<T, __half>::value) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t y;
  if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}

// Quantises a row that kLanes neighbouring lanes hold together (8 16-bit values per lane, all lanes of the group active).
// Returns the lane's 8 codes as 4 bytes; `params` (scale in the low half, offset in the high half) is the same on every
// lane of the group.  Values beyond the clamp need no clamp of their own: their code lies beyond 0 or 15 and is clamped.
// A code becomes an integer by adding 1.5 * 2^23 (round to nearest even, as rint), and the eight are put together by
// multiply-adds modulo 2^32, from which the constants' sum is taken off: the conversion and shift units stay free.
template <typename T, int kLanes>
__device__ __forceinline__ uint32_t int4_quantise(uint4 raw, bool odd_slot, uint32_t& params) {
  // smallest and (negated) largest value side by side
  const uint32_t small = min2_nan<T>(min2_nan<T>(raw.x, raw.y), min2_nan<T>(raw.z, raw.w));
  const uint32_t large = max2_nan<T>(max2_nan<T>(raw.x, raw.y), max2_nan<T>(raw.z, raw.w)) ^ 0x80008000u;
  uint32_t ends = min2_nan<T>(__byte_perm(small, large, 0x5410), __byte_perm(small, large, 0x7632));
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) ends = min2_nan<T>(ends, __shfl_xor_sync(0xffffffffu, ends, o));
  const float2 both = unpack2<T>(ends);
  float lo = both.x, hi = -both.y;
  float x[8];
  {
    const float2 a = unpack2<T>(raw.x), b = unpack2<T>(raw.y), c = unpack2<T>(raw.z), d = unpack2<T>(raw.w);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
  }
  lo = min_nan(max_nan(lo, -kInt4Clamp), kInt4Clamp);
  hi = min_nan(max_nan(hi, -kInt4Clamp), kInt4Clamp);
  // (hi - lo) / 15, correctly rounded: Markstein's step with the correctly rounded 1 / 15 (where it underflows the float16
  // is 0 either way)
  const float span = hi - lo;
  constexpr float kFifteenth = 1.f / 15.f;
  const float rough = __fmul_rn(span, kFifteenth);
  const __half step = __float2half_rn(fmaf(fmaf(-15.f, rough, span), kFifteenth, rough));
  const __half scale = odd_slot ? __hneg(step) : step;
  const __half offset = __float2half_rn(odd_slot ? hi : lo);
  const float s = __half2float(scale), m = __half2float(offset);
  const float inverse = s == 0.f ? 0.f : __frcp_rn(s);
  constexpr float kMagic = 12582912.f;
  constexpr uint32_t kMagicBits = 0x4b400000u;
  // Codes stay between 0 and 15 by themselves unless the scale is a subnormal, an end was rounded or clamped, or the row has
  // a NaN: the scale's rounding moves 15 steps by 15 x 2^-11 of one.
  const bool plain = fabsf(s) >= 6.103515625e-5f && m == (odd_slot ? hi : lo) && lo > -kInt4Clamp && hi < kInt4Clamp;
  uint32_t codes = 0;
  if (__all_sync(0xffffffffu, plain)) {
#pragma unroll
    for (int e = 7; e >= 0; --e) codes = codes * 16u + __float_as_uint(__fadd_rn(__fmul_rn(x[e] - m, inverse), kMagic));
  } else {
#pragma unroll
    for (int e = 7; e >= 0; --e) {
      const float c = fminf(fmaxf(__fmul_rn(x[e] - m, inverse), 0.f), 15.f);   // a NaN becomes 0
      codes = codes * 16u + __float_as_uint(__fadd_rn(c, kMagic));
    }
  }
  params = uint32_t(__half_as_ushort(scale)) | (uint32_t(__half_as_ushort(offset)) << 16);
  return codes - kMagicBits * 0x11111111u;
}

}  // namespace tb200
