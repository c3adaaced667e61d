// Per-head RMS norm of q and k with the GPT-NeoX rotation in the same pass, and the append of k and v to a paged cache
// (16-bit, or 4 bits with one scale and offset per token and KV head) in the same launch, sm_100a.
//
// Per row x of D values (one token, one head):
//   y = x * rsqrt(mean(x^2) + eps) * w
//   z1 = y1 cos a - y2 sin a, z2 = y2 cos a + y1 sin a   for the halves (y1, y2) of the first rotary_dim values,
//   a_j = position * inv_freq_j
// all in fp32 and rounded ONCE, to the 16-bit output.  v rows are copied (or quantised) as they are.  The 4-bit cache
// gets k from its 16-bit rounded value, so that append and fused append agree bit for bit.
//
// The angle is computed here rather than read from a cos / sin table: position * inv_freq / 2 pi in fp64 (a far position
// times a frequency has more digits than fp32 holds), reduced to a fraction of a turn, then one sincospif per (token,
// frequency) shared by all heads through shared memory.  No table means no largest position and no gathers.
//
// HBM bound: every row is read and written once.  A group of lanes holds a row, 8 values each, and requests four rows
// before it works on the first, while the block's angles are still being computed; where all dims rotate, a lane's values are
// 4 of the first half and their 4 partners, so that the rotation needs no shuffles.  Measured, 8192 tokens of 32 / 8 heads x
// 128, bf16: with the append to a 16-bit cache 41 us = 4.9 TB/s (copies run at 6.5); the SMs issue 64 % of the time and
// warps wait for their rows and for the schedulers alike.  The 4-bit append of 11755 tokens of 8 heads takes 28 us = 2.2
// TB/s: about 200 instructions for 8 values of a row, a third of them for its two parameters.
#include <type_traits>

#include "int4_cache.cuh"

namespace tb200 {
namespace {

constexpr int kThreads = 128;
enum CacheKind { kNoCache = 0, kCache16 = 1, kCacheInt4 = 2 };

struct RowsParams {
  const void *q, *k, *v;
  void *q_out, *k_out;
  const void *q_weight, *k_weight;   // NULL: ones
  int weight_f32;
  const double* inv_turns;           // [rotary_dim / 2]: inv_freq / 2 pi
  const int32_t* positions;
  const int32_t* slots;
  void *k_cache, *v_cache;           // kCacheInt4: k_cache is the one pool
  int heads, heads_kv, dim, rotary_dim, page_size;
  int rows;                          // rows of a token: q heads, k heads, then v heads when there is a cache
  int q_tok, q_head, k_tok, k_head, v_tok, v_head;       // strides in elements
  unsigned by_heads, by_heads_kv, by_half;               // reciprocals for the divisions by heads, heads_kv and rotary_dim / 2
  int pool_tokens, tokens, block_tokens;
  float eps, inv_dim;
};

// The 8 values of a lane: consecutive ones, or (kSplit) 4 at `at` and 4 at `at + half`.
template <typename T, bool kSplit>
__device__ __forceinline__ uint4 load_row(const T* p, int half) {
  if constexpr (!kSplit) return __ldg(reinterpret_cast<const uint4*>(p));
  const uint2 a = __ldg(reinterpret_cast<const uint2*>(p)), b = __ldg(reinterpret_cast<const uint2*>(p + half));
  return make_uint4(a.x, a.y, b.x, b.y);
}
template <typename T, bool kSplit>
__device__ __forceinline__ void store_row(T* p, int half, uint4 v) {
  if constexpr (!kSplit) {
    *reinterpret_cast<uint4*>(p) = v;
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(v.x, v.y);
    *reinterpret_cast<uint2*>(p + half) = make_uint2(v.z, v.w);
  }
}
template <typename T>
__device__ __forceinline__ void unpack8(uint4 u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}
// Weights of a lane's values (element e at at + e, from e = 4 on at at2 + e - 4), kept in 16 bits where they come so.
template <typename T>
__device__ __forceinline__ void load_weight8(const void* w, int f32, int at, int at2, bool active, float (&x)[8]) {
  if (!w || !active) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 1.f;
    return;
  }
  if (!f32 && (reinterpret_cast<uintptr_t>(w) & 7) == 0) {
    const uint2 a = __ldg(reinterpret_cast<const uint2*>(static_cast<const T*>(w) + at));
    const uint2 b = __ldg(reinterpret_cast<const uint2*>(static_cast<const T*>(w) + at2));
    unpack8<T>(make_uint4(a.x, a.y, b.x, b.y), x);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = e < 4 ? at + e : at2 + e - 4;
    x[e] = f32 ? __ldg(static_cast<const float*>(w) + d) : float(static_cast<const T*>(w)[d]);
  }
}

constexpr int kMaxTokens = 8;      // of a block

// n / d for n < 2^16 by the reciprocal 2^32 / d, rounded up (0 where d is 1)
inline unsigned reciprocal(int d) { return d <= 1 ? 0u : 0xffffffffu / unsigned(d) + 1u; }
__device__ __forceinline__ int divide(int n, unsigned by) { return by ? int(__umulhi(unsigned(n), by)) : n; }
enum RowKind { kRowQ = 0, kRowK = 1, kRowV = 2 };

// A block of `block_tokens` tokens; kLanes lanes hold a row, 8 values each.  q, k and v rows are walked one kind after the
// other, so that weights, pointers and what becomes of a row are settled outside the loop over rows.  With the norm eight
// blocks share an SM, 64 registers a thread (with the 4-bit append and read-back of 8192 tokens 60.8 us against 63.2).
template <typename T, int kLanes, int kCache, bool kNorm, bool kSplit>
__global__ void __launch_bounds__(kThreads, kNorm ? 8 : 1) rows_kernel(RowsParams p) {
  constexpr int kGroups = kThreads / kLanes;
  extern __shared__ float2 s_turn[];       // [block_tokens][half]: cos, sin
  // where the tokens' rows go: element (16-bit cache) or byte of the record (4-bit) of head 0, -1: nowhere; row of the record
  __shared__ long long s_to[kMaxTokens];
  __shared__ int s_row[kMaxTokens];
  const int t0 = blockIdx.x * p.block_tokens;
  const int n_tokens = min(p.block_tokens, p.tokens - t0);
  const int lane = threadIdx.x & (kLanes - 1), group = threadIdx.x / kLanes;
  const int half = p.rotary_dim >> 1;
  const int at = kSplit ? lane * 4 : lane * 8, at2 = kSplit ? half + lane * 4 : at + 4;   // first and fifth value
  const bool active = kSplit ? at < half : at < p.dim;
  const long long head_bytes = (long long)(p.page_size / kInt4Tokens) * int4_record_bytes(p.dim);
  bool ready = false;

  // angles and destinations of the block's tokens, worked out while the first rows are on their way
  auto prepare = [&] {
    if (kCache != kNoCache && threadIdx.x < n_tokens) {
      const int slot = p.slots[t0 + threadIdx.x];
      long long to = -1;
      if (slot >= 0 && slot < p.pool_tokens) {
        if constexpr (kCache == kCacheInt4) {
          const int page = slot / p.page_size, off = slot - page * p.page_size;
          to = (long long)page * p.heads_kv * head_bytes + (long long)(off / kInt4Tokens) * int4_record_bytes(p.dim);
          s_row[threadIdx.x] = off % kInt4Tokens;      // a record begins at an even slot: the parity is the slot's
        } else {
          to = (long long)slot * p.heads_kv * p.dim;
        }
      }
      s_to[threadIdx.x] = to;
    }
    if constexpr (kNorm) {
      for (int j = threadIdx.x; j < n_tokens * half; j += kThreads) {
        const int tt = n_tokens == 1 ? 0 : divide(j, p.by_half);
        const double turns = double(p.positions[t0 + tt]) * p.inv_turns[j - tt * half];
        float s, c;
        sincospif(2.f * float(turns - rint(turns)), &s, &c);
        s_turn[j] = make_float2(c, s);
      }
    }
    __syncthreads();
  };

  // kAhead rows of one kind, from item i0 (token of the block * rows + row) in steps of kGroups
  auto walk = [&](auto kind_, auto ahead_, const T* src, int tok_stride, int head_stride, int rows, unsigned by_rows,
                  const void* weight) {
    constexpr int kKind = decltype(kind_)::value, kAhead = decltype(ahead_)::value;
    constexpr bool kNormed = kNorm && kKind != kRowV;
    const int items = n_tokens * rows;
    src += (long long)t0 * tok_stride + at;
    T* out_rows = static_cast<T*>(kKind == kRowQ ? p.q_out : kKind == kRowK ? p.k_out : nullptr);
    if (out_rows) out_rows += (long long)t0 * rows * p.dim + at;
    float w[8];
    for (int i0 = group; i0 - group < items; i0 += kGroups * kAhead) {      // the lanes of a warp stay together
      uint4 raw[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int item = i0 + a * kGroups;
        raw[a] = make_uint4(0u, 0u, 0u, 0u);
        if (item < items && active) {
          const int tt = n_tokens == 1 ? 0 : divide(item, by_rows), r = item - tt * rows;
          raw[a] = load_row<T, kSplit>(src + (long long)tt * tok_stride + (long long)r * head_stride, half);
        }
      }
      if constexpr (kNormed) {
        if (i0 == group) load_weight8<T>(weight, p.weight_f32, at, at2, active, w);
      }
      if (!ready) {
        ready = true;
        prepare();
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int item = i0 + a * kGroups;
        if (item - group >= items) break;          // the same for the whole block
        const bool live = item < items;            // a group behind the last row only takes part in the shuffles
        const int tt = n_tokens == 1 || !live ? 0 : divide(item, by_rows), r = live ? item - tt * rows : 0;
        uint4 out = raw[a];
        if constexpr (kNormed) {
          float x[8];
          unpack8<T>(raw[a], x);
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
          for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float inv = rsqrtf(fmaf(sum, p.inv_dim, p.eps));
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = x[e] * inv * w[e];
          const float2* turn = s_turn + tt * half;
          if constexpr (kSplit) {
            const int j = active ? at : 0;      // lanes behind the row have no angles
            const float4 cs0 = *reinterpret_cast<const float4*>(turn + j), cs1 = *reinterpret_cast<const float4*>(turn + j + 2);
            const float c[4] = {cs0.x, cs0.z, cs1.x, cs1.z}, s[4] = {cs0.y, cs0.w, cs1.y, cs1.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[e] = y[e] * c[e] - y[e + 4] * s[e];
              x[e + 4] = y[e + 4] * c[e] + y[e] * s[e];
            }
          } else {
            const bool first = at < half, rotated = at < p.rotary_dim;
            const int partner = rotated ? (first ? lane + half / 8 : lane - half / 8) : lane;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float other = __shfl_sync(0xffffffffu, y[e], partner, kLanes);
              x[e] = y[e];
              if (rotated) {
                const float2 cs = turn[(first ? at : at - half) + e];
                x[e] = first ? y[e] * cs.x - other * cs.y : y[e] * cs.x + other * cs.y;
              }
            }
          }
          out = pack8<T>(x);
        }
        if (out_rows && live && active) store_row<T, kSplit>(out_rows + (long long)item * p.dim, half, out);
        if constexpr (kKind != kRowQ && kCache == kCache16) {
          const long long to = live ? s_to[tt] : -1;
          if (to >= 0 && active)
            store_row<T, kSplit>(static_cast<T*>(kKind == kRowK ? p.k_cache : p.v_cache) + to + r * p.dim + at, half, out);
        }
        if constexpr (kKind != kRowQ && kCache == kCacheInt4) {
          const long long to = live ? s_to[tt] : -1;
          const int tok = live ? s_row[tt] : 0;
          uint32_t params;
          const uint32_t codes = int4_quantise<T, kLanes>(out, tok & 1, params);
          if (to >= 0) {
            constexpr int part = kKind == kRowK ? 0 : 1;
            unsigned char* rec = static_cast<unsigned char*>(p.k_cache) + to + r * head_bytes;
            unsigned char* row = rec + (part * kInt4Tokens + tok) * (p.dim / 2);
            if constexpr (kSplit) {
              *reinterpret_cast<uint16_t*>(row + lane * 2) = uint16_t(codes);
              *reinterpret_cast<uint16_t*>(row + p.dim / 4 + lane * 2) = uint16_t(codes >> 16);
            } else {
              *reinterpret_cast<uint32_t*>(row + lane * 4) = codes;
            }
            if (lane == 0) *reinterpret_cast<uint32_t*>(rec + kInt4Tokens * p.dim + tok * 8 + part * 4) = params;
          }
        }
      }
    }
  };
  using Q = std::integral_constant<int, kRowQ>;
  using K = std::integral_constant<int, kRowK>;
  using V = std::integral_constant<int, kRowV>;
  using Ahead = std::integral_constant<int, 4>;
  if constexpr (kNorm)
    walk(Q{}, Ahead{}, static_cast<const T*>(p.q), p.q_tok, p.q_head, p.heads, p.by_heads, p.q_weight);
  walk(K{}, Ahead{}, static_cast<const T*>(p.k), p.k_tok, p.k_head, p.heads_kv, p.by_heads_kv, p.k_weight);
  if constexpr (kCache != kNoCache)
    walk(V{}, Ahead{}, static_cast<const T*>(p.v), p.v_tok, p.v_head, p.heads_kv, p.by_heads_kv, nullptr);
}

template <typename T, int kLanes, int kCache, bool kNorm>
void launch_lanes(RowsParams p, int tokens, cudaStream_t s) {
  constexpr int kGroups = kThreads / kLanes;
  p.tokens = tokens;
  p.inv_dim = 1.f / float(p.dim);
  p.by_heads = reciprocal(p.heads);
  p.by_heads_kv = reciprocal(p.heads_kv);
  p.by_half = reciprocal(p.rotary_dim / 2);
  // about kRowsPerGroup rows for every group of lanes, however few heads there are
  constexpr int kRowsPerGroup = 12;
  p.block_tokens = kRowsPerGroup * kGroups / p.rows;
  if (p.block_tokens < 1) p.block_tokens = 1;
  if (p.block_tokens > kMaxTokens) p.block_tokens = kMaxTokens;
  // but three blocks for every SM where there are as many tokens (with the 4-bit append and read-back of 2047 tokens of 16 / 4
  // heads x 64: 10 us in 512 blocks, 11 in 256, 17 in 2047; 8192 of 32 / 8 heads x 128 into a 16-bit cache: 41 us with two
  // tokens a block, 46 with one)
  while (p.block_tokens > 1 && tokens / p.block_tokens < sm_count() * 3) --p.block_tokens;
  const int blocks = (tokens + p.block_tokens - 1) / p.block_tokens;
  const size_t smem = kNorm ? size_t(p.block_tokens) * (p.rotary_dim / 2) * sizeof(float2) : 0;
  if (kNorm && p.rotary_dim == p.dim && p.dim % 16 == 0)
    rows_kernel<T, kLanes, kCache, kNorm, kNorm><<<blocks, kThreads, smem, s>>>(p);
  else
    rows_kernel<T, kLanes, kCache, kNorm, false><<<blocks, kThreads, smem, s>>>(p);
}
template <typename T, int kCache, bool kNorm>
void launch_rows(const RowsParams& p, int tokens, cudaStream_t s) {
  if (p.dim <= 64)
    launch_lanes<T, 8, kCache, kNorm>(p, tokens, s);
  else if (p.dim <= 128)
    launch_lanes<T, 16, kCache, kNorm>(p, tokens, s);
  else if constexpr (kCache != kCacheInt4)
    launch_lanes<T, 32, kCache, kNorm>(p, tokens, s);
}

// 16-byte rows: the base and both strides
bool aligned_rows(const void* base, int64_t tok, int64_t head) {
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && tok % 8 == 0 && head % 8 == 0;
}
bool fits_int(int64_t stride) { return stride >= -0x7fffffffLL && stride <= 0x7fffffffLL; }
constexpr int kMaxHeads = 4096;     // (token, row) pairs of a block are divided in 16 bits

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" int tb200_qk_norm_rope(const void* q, const void* k, const void* v, void* q_out, void* k_out,
                                  const void* q_weight, const void* k_weight, int weight_dtype, const double* inv_turns,
                                  const int32_t* positions, const int32_t* slots, void* k_cache, void* v_cache,
                                  int dtype, int cache, int tokens, int heads, int heads_kv, int dim, int rotary_dim,
                                  int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                                  int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, int page_size,
                                  int64_t pool_tokens, float eps, void* stream) {
  if (tokens < 0 || heads <= 0 || heads_kv <= 0 || dim <= 0)
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "heads, heads_kv and dim must be positive and tokens not negative");
  if (dtype != TB200_BF16 && dtype != TB200_F16) TB200_FAIL(TB200_ERR_UNSUPPORTED, "dtype must be F16 or BF16");
  if (dim % 8 != 0 || dim > 256) TB200_FAIL(TB200_ERR_UNSUPPORTED, "head dim must be a multiple of 8 up to 256, got %d", dim);
  if (rotary_dim < 0 || rotary_dim > dim || rotary_dim % 16 != 0)
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "rotary_dim must be a multiple of 16 up to the head dim, got %d", rotary_dim);
  if (cache < TB200_CACHE_NONE || cache > TB200_CACHE_INT4) TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "unknown kind of cache");
  if (weight_dtype != dtype && weight_dtype != TB200_F32)
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "weights must have the dtype of q or be F32");
  if (cache == TB200_CACHE_INT4) {
    if (dim != 64 && dim != 128) TB200_FAIL(TB200_ERR_UNSUPPORTED, "a 4-bit cache serves head dim 64 and 128, got %d", dim);
    if (page_size <= 0 || page_size % kInt4Tokens != 0)
      TB200_FAIL(TB200_ERR_UNSUPPORTED, "page_size must be a multiple of 16, got %d", page_size);
  }
  if (pool_tokens < 0 || pool_tokens > 0x7fffffffLL) TB200_FAIL(TB200_ERR_UNSUPPORTED, "the pool must hold fewer than 2^31 tokens");
  if (tokens > 1 << 30) TB200_FAIL(TB200_ERR_UNSUPPORTED, "at most 2^30 tokens");    // rows are counted in 32 bits
  if (tokens == 0) return TB200_OK;
  if (!q || !k || !q_out || !positions || (rotary_dim > 0 && !inv_turns))
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "q, k, q_out, positions and inv_turns must be non-null");
  if (cache != TB200_CACHE_NONE && (!v || !slots || !k_cache || (cache == TB200_CACHE_16BIT && !v_cache)))
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "v, slots and the cache must be non-null");
  if (!aligned_rows(q, q_token_stride, q_head_stride) || !aligned_rows(k, k_token_stride, k_head_stride) ||
      !aligned_rows(q_out, 0, 0) || !aligned_rows(k_out, 0, 0) ||
      (cache != TB200_CACHE_NONE && (!aligned_rows(v, v_token_stride, v_head_stride) || !aligned_rows(k_cache, 0, 0) ||
                                     !aligned_rows(v_cache, 0, 0))))
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "rows must start on 16-byte boundaries");
  if (heads > kMaxHeads || heads_kv > kMaxHeads) TB200_FAIL(TB200_ERR_UNSUPPORTED, "at most %d heads", kMaxHeads);
  if (!fits_int(q_token_stride) || !fits_int(q_head_stride) || !fits_int(k_token_stride) || !fits_int(k_head_stride) ||
      !fits_int(v_token_stride) || !fits_int(v_head_stride))
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "strides must fit 32 bits");
  RowsParams p{};
  p.q = q; p.k = k; p.v = v; p.q_out = q_out; p.k_out = k_out;
  p.q_weight = q_weight; p.k_weight = k_weight; p.weight_f32 = weight_dtype == TB200_F32;
  p.inv_turns = inv_turns; p.positions = positions; p.slots = slots; p.k_cache = k_cache; p.v_cache = v_cache;
  p.heads = heads; p.heads_kv = heads_kv; p.dim = dim; p.rotary_dim = rotary_dim; p.page_size = page_size;
  p.rows = heads + heads_kv + (cache != TB200_CACHE_NONE ? heads_kv : 0);
  p.q_tok = int(q_token_stride); p.q_head = int(q_head_stride); p.k_tok = int(k_token_stride);
  p.k_head = int(k_head_stride); p.v_tok = int(v_token_stride); p.v_head = int(v_head_stride);
  p.pool_tokens = int(pool_tokens); p.eps = eps;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TB200_BF16) {
    if (cache == TB200_CACHE_NONE) launch_rows<__nv_bfloat16, kNoCache, true>(p, tokens, s);
    else if (cache == TB200_CACHE_16BIT) launch_rows<__nv_bfloat16, kCache16, true>(p, tokens, s);
    else launch_rows<__nv_bfloat16, kCacheInt4, true>(p, tokens, s);
  } else {
    if (cache == TB200_CACHE_NONE) launch_rows<__half, kNoCache, true>(p, tokens, s);
    else if (cache == TB200_CACHE_16BIT) launch_rows<__half, kCache16, true>(p, tokens, s);
    else launch_rows<__half, kCacheInt4, true>(p, tokens, s);
  }
  TB200_CUDA_CHECK(cudaGetLastError());
  return TB200_OK;
}

extern "C" int tb200_int4_cache_append(const void* k, const void* v, const int32_t* slots, void* kv_pages, int dtype,
                                       int tokens, int heads_kv, int dim, int page_size, int64_t pool_tokens,
                                       int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                                       int64_t v_head_stride, void* stream) {
  if (tokens < 0 || heads_kv <= 0) TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "heads_kv must be positive and tokens not negative");
  if (dtype != TB200_BF16 && dtype != TB200_F16) TB200_FAIL(TB200_ERR_UNSUPPORTED, "dtype must be F16 or BF16");
  if (dim != 64 && dim != 128) TB200_FAIL(TB200_ERR_UNSUPPORTED, "a 4-bit cache serves head dim 64 and 128, got %d", dim);
  if (page_size <= 0 || page_size % kInt4Tokens != 0)
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "page_size must be a multiple of 16, got %d", page_size);
  if (pool_tokens < 0 || pool_tokens > 0x7fffffffLL) TB200_FAIL(TB200_ERR_UNSUPPORTED, "the pool must hold fewer than 2^31 tokens");
  if (tokens > 1 << 30) TB200_FAIL(TB200_ERR_UNSUPPORTED, "at most 2^30 tokens");    // rows are counted in 32 bits
  if (tokens == 0) return TB200_OK;
  if (!k || !v || !slots || !kv_pages) TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "k, v, slots and kv_pages must be non-null");
  if (!aligned_rows(k, k_token_stride, k_head_stride) || !aligned_rows(v, v_token_stride, v_head_stride) ||
      !aligned_rows(kv_pages, 0, 0))
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "rows must start on 16-byte boundaries");
  if (heads_kv > kMaxHeads) TB200_FAIL(TB200_ERR_UNSUPPORTED, "at most %d heads", kMaxHeads);
  if (!fits_int(k_token_stride) || !fits_int(k_head_stride) || !fits_int(v_token_stride) || !fits_int(v_head_stride))
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "strides must fit 32 bits");
  RowsParams p{};
  p.k = k; p.v = v; p.slots = slots; p.k_cache = kv_pages;
  p.heads = 0; p.heads_kv = heads_kv; p.dim = dim; p.page_size = page_size; p.rows = 2 * heads_kv;
  p.k_tok = int(k_token_stride); p.k_head = int(k_head_stride); p.v_tok = int(v_token_stride); p.v_head = int(v_head_stride);
  p.pool_tokens = int(pool_tokens);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TB200_BF16) launch_rows<__nv_bfloat16, kCacheInt4, false>(p, tokens, s);
  else launch_rows<__half, kCacheInt4, false>(p, tokens, s);
  TB200_CUDA_CHECK(cudaGetLastError());
  return TB200_OK;
}
