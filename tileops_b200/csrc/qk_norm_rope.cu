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
// HBM bound: every row is read and written once.
#include "int4_cache.cuh"

namespace tb200 {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxHalf = 128;      // rotary_dim / 2
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
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;   // strides in elements
  int pool_tokens;
  float eps;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
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
template <typename T>
__device__ __forceinline__ void load_weight8(const void* w, int f32, int at, bool active, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 1.f;
  if (!w || !active) return;
  if (f32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = static_cast<const float*>(w)[at + e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = float(static_cast<const T*>(w)[at + e]);
  }
}

// One block per token; kLanes lanes hold a row, 8 values each.
template <typename T, int kLanes, int kCache, bool kNorm>
__global__ void __launch_bounds__(kThreads) rows_kernel(RowsParams p) {
  __shared__ float2 s_turn[kMaxHalf];
  const int t = blockIdx.x;
  const int lane = threadIdx.x & (kLanes - 1);
  const int group = threadIdx.x / kLanes;
  constexpr int kGroups = kThreads / kLanes;
  const int at = lane * 8;
  const bool active = at < p.dim;
  const int half = p.rotary_dim >> 1;
  float wq[8], wk[8];
  if constexpr (kNorm) {
    const double pos = double(p.positions[t]);
    for (int j = threadIdx.x; j < half; j += kThreads) {
      const double turns = pos * p.inv_turns[j];
      float s, c;
      sincospif(2.f * float(turns - rint(turns)), &s, &c);
      s_turn[j] = make_float2(c, s);
    }
    load_weight8<T>(p.q_weight, p.weight_f32, at, active, wq);
    load_weight8<T>(p.k_weight, p.weight_f32, at, active, wk);
    __syncthreads();
  }
  const int slot = kCache != kNoCache ? p.slots[t] : -1;
  const bool stored = slot >= 0 && slot < p.pool_tokens;

  for (int r0 = 0; r0 < p.rows; r0 += kGroups) {      // all lanes of a warp stay together for the shuffles
    const int r = r0 + group;
    const bool live = r < p.rows;
    const bool is_q = r < p.heads, is_k = !is_q && r < p.heads + p.heads_kv;
    const int h = is_q ? r : is_k ? r - p.heads : r - p.heads - p.heads_kv;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live && active) {
      const T* src = is_q   ? static_cast<const T*>(p.q) + t * p.q_tok + h * p.q_head
                     : is_k ? static_cast<const T*>(p.k) + t * p.k_tok + h * p.k_head
                            : static_cast<const T*>(p.v) + t * p.v_tok + h * p.v_head;
      load8(src + at, x);
    }
    if constexpr (kNorm) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const bool normed = is_q || is_k;
      const float inv = rsqrtf(sum / float(p.dim) + p.eps);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = normed ? x[e] * inv * (is_q ? wq[e] : wk[e]) : x[e];
      const bool first = at < half, rotated = at < p.rotary_dim;
      const int partner = rotated ? (first ? lane + half / 8 : lane - half / 8) : lane;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl_sync(0xffffffffu, y[e], partner, kLanes);
        x[e] = y[e];
        if (rotated && normed) {
          const float2 cs = s_turn[(first ? at : at - half) + e];
          x[e] = first ? y[e] * cs.x - other * cs.y : y[e] * cs.x + other * cs.y;
        }
      }
    }
    const uint4 out = pack8<T>(x);
    if (live && active) {
      if (is_q) {
        if (p.q_out) *reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + (size_t(t) * p.heads + h) * p.dim + at) = out;
      } else if (is_k && p.k_out) {
        *reinterpret_cast<uint4*>(static_cast<T*>(p.k_out) + (size_t(t) * p.heads_kv + h) * p.dim + at) = out;
      }
    }
    if constexpr (kCache == kCache16) {
      if (live && active && !is_q && stored) {
        T* pool = static_cast<T*>(is_k ? p.k_cache : p.v_cache);
        *reinterpret_cast<uint4*>(pool + (size_t(slot) * p.heads_kv + h) * p.dim + at) = out;
      }
    }
    if constexpr (kCache == kCacheInt4) {
      float z[8];
      const uint32_t w[4] = {out.x, out.y, out.z, out.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(w[i]);
        z[2 * i] = f.x;
        z[2 * i + 1] = f.y;
      }
      uint32_t params;
      const uint32_t codes = int4_quantise<kLanes>(z, slot & 1, params);
      if (live && !is_q && stored) {
        unsigned char* rec = static_cast<unsigned char*>(p.k_cache) +
                             int4_record_of(slot, h, p.heads_kv, p.page_size, p.dim);
        const int tok = slot % kInt4Tokens;
        const int part = is_k ? 0 : 1;
        *reinterpret_cast<uint32_t*>(rec + (part * kInt4Tokens + tok) * (p.dim / 2) + lane * 4) = codes;
        if (lane == 0) *reinterpret_cast<uint32_t*>(rec + kInt4Tokens * p.dim + tok * 8 + part * 4) = params;
      }
    }
  }
}

template <typename T, int kCache, bool kNorm>
void launch_rows(const RowsParams& p, int tokens, cudaStream_t s) {
  if (p.dim <= 64)
    rows_kernel<T, 8, kCache, kNorm><<<tokens, kThreads, 0, s>>>(p);
  else if (p.dim <= 128)
    rows_kernel<T, 16, kCache, kNorm><<<tokens, kThreads, 0, s>>>(p);
  else if constexpr (kCache != kCacheInt4)
    rows_kernel<T, 32, kCache, kNorm><<<tokens, kThreads, 0, s>>>(p);
}

// 16-byte rows: the base and both strides
bool aligned_rows(const void* base, int64_t tok, int64_t head) {
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && tok % 8 == 0 && head % 8 == 0;
}

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
  RowsParams p{};
  p.q = q; p.k = k; p.v = v; p.q_out = q_out; p.k_out = k_out;
  p.q_weight = q_weight; p.k_weight = k_weight; p.weight_f32 = weight_dtype == TB200_F32;
  p.inv_turns = inv_turns; p.positions = positions; p.slots = slots; p.k_cache = k_cache; p.v_cache = v_cache;
  p.heads = heads; p.heads_kv = heads_kv; p.dim = dim; p.rotary_dim = rotary_dim; p.page_size = page_size;
  p.rows = heads + heads_kv + (cache != TB200_CACHE_NONE ? heads_kv : 0);
  p.q_tok = q_token_stride; p.q_head = q_head_stride; p.k_tok = k_token_stride; p.k_head = k_head_stride;
  p.v_tok = v_token_stride; p.v_head = v_head_stride;
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
  if (tokens == 0) return TB200_OK;
  if (!k || !v || !slots || !kv_pages) TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "k, v, slots and kv_pages must be non-null");
  if (!aligned_rows(k, k_token_stride, k_head_stride) || !aligned_rows(v, v_token_stride, v_head_stride) ||
      !aligned_rows(kv_pages, 0, 0))
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "rows must start on 16-byte boundaries");
  RowsParams p{};
  p.k = k; p.v = v; p.slots = slots; p.k_cache = kv_pages;
  p.heads = 0; p.heads_kv = heads_kv; p.dim = dim; p.page_size = page_size; p.rows = 2 * heads_kv;
  p.k_tok = k_token_stride; p.k_head = k_head_stride; p.v_tok = v_token_stride; p.v_head = v_head_stride;
  p.pool_tokens = int(pool_tokens);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TB200_BF16) launch_rows<__nv_bfloat16, kCacheInt4, false>(p, tokens, s);
  else launch_rows<__half, kCacheInt4, false>(p, tokens, s);
  TB200_CUDA_CHECK(cudaGetLastError());
  return TB200_OK;
}
