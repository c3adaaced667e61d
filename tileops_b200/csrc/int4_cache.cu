// Reads a 4-bit paged KV cache back as packed 16-bit K and V, sm_100a: the cache side of a chunked prefill, whose
// tcgen05 attention kernel takes 16-bit operands.  value = scale * code + offset in fp32 (the product is exact), rounded
// once (float16: saturated at +-65504).  HBM bound: dim + 8 bytes read and 4 dim written per token and KV head.
#include "int4_cache.cuh"

namespace tb200 {
namespace {

constexpr int kThreads = 256;

struct GatherParams {
  const unsigned char* pages;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* cu;        // [batch + 1]: request b owns output rows cu[b] .. cu[b + 1]
  const int32_t* cached;    // NULL: all of a request's rows are cached; else its first cached[b] rows
  const int32_t* cu_new;    // rows behind the cached ones come from k_new / v_new, request b from row cu_new[b] on
  const void *k_new, *v_new;
  void *k_out, *v_out;
  int batch, heads_kv, page_size, table_width, pool_pages, total;
};

// Blocks walk over pieces of kTokens output rows (tokens).  One warp finds where the tokens of the next piece come from (a
// binary search and a block-table entry each, four dependent reads and more) while eight expand the rows of this one:
// D / 16 lanes hold a row of one token and KV head, 8 values of each half, so that a store fills whole sectors (16 values
// in a row each: 87 against 80 us for the read-back and append of 52 thousand tokens, 8 heads x 128); neighbouring groups
// take neighbouring tokens, whose rows lie next to each other in a record.  kAhead rows are requested before the first is
// expanded.  Short pieces spread few tokens over more blocks and leave less of the last round idle: read-back and append of
// 449 tokens 6.5 / 7.6 / 9.9 us with 8 / 16 / 32 tokens a piece, of the 52 thousand 75.5 / 75.5 / 79.2 us.
constexpr int kTokens = 8;
constexpr int kAhead = 4;
constexpr int kBlocksPerSm = 5;

// Two values side by side.  15 steps between +-65504 end 32 beyond the largest float16 (their scale is rounded to 8736): a
// float16 read-back saturates, as the append does.  bfloat16 holds them.
template <typename T>
__device__ __forceinline__ uint32_t pack_value(float a, float b) {
  const uint32_t v = pack2<T>(a, b);
  if constexpr (std::is_same<T, __half>::value) return max2_nan<T>(min2_nan<T>(v, 0x7bff7bffu), 0xfbfffbffu);
  return v;
}

// The rows of one piece, by the kThreads working threads.
template <typename T, int D>
__device__ __forceinline__ void expand(const GatherParams& p, int g0, const long long* s_src, const int* s_row,
                                       long long head_bytes) {
  constexpr int kLanes = D / 16;
  constexpr int kGroups = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int items = 2 * p.heads_kv * kTokens;     // (K or V, head, token), tokens fastest
  for (int i0 = group; i0 < items; i0 += kGroups * kAhead) {
    uint2 codes[kAhead];
    uint32_t params[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int item = i0 + a * kGroups;
      codes[a] = make_uint2(0u, 0u);
      params[a] = 0x7e007e00u;
      if (item >= items) continue;
      const int tok = item % kTokens, row = item / kTokens, h = row >> 1, part = row & 1;
      const long long src = s_src[tok];
      if (src >= 0) {
        const unsigned char* rec = p.pages + src + h * head_bytes;
        const int r = s_row[tok];
        const unsigned char* row = rec + (part * kInt4Tokens + r) * (D / 2) + lane * 4;
        codes[a].x = __ldg(reinterpret_cast<const uint32_t*>(row));
        codes[a].y = __ldg(reinterpret_cast<const uint32_t*>(row + D / 4));
        params[a] = __ldg(reinterpret_cast<const uint32_t*>(rec + kInt4Tokens * D + r * 8 + part * 4));
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int item = i0 + a * kGroups;
      if (item >= items) continue;
      const int tok = item % kTokens, row = item / kTokens, h = row >> 1, part = row & 1;
      const long long src = s_src[tok];
      if (src == -2) continue;
      const size_t to = (size_t(g0 + tok) * p.heads_kv + h) * D + lane * 8;
      uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(part ? p.v_out : p.k_out) + to);
      if (src <= -3) {
        const size_t from = (size_t(-3 - src) * p.heads_kv + h) * D + lane * 8;
        const uint4* in = reinterpret_cast<const uint4*>(static_cast<const T*>(part ? p.v_new : p.k_new) + from);
        out[0] = __ldg(in);
        out[D / 16] = __ldg(in + D / 16);
        continue;
      }
      // a nibble masked into the low bits of a float16 is the number c * 2^-24: two codes per mask, no conversion
      const float2 sm = f16x2_to_f32x2(params[a]);
      const float lo = sm.x * 16777216.f, hi = sm.x * 1048576.f, m = sm.y;
      const uint32_t c[2] = {codes[a].x, codes[a].y};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x[8];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const uint32_t v = b ? c[i] >> 8 : c[i];
          const float2 even = f16x2_to_f32x2(v & 0x000f000fu), odd = f16x2_to_f32x2(v & 0x00f000f0u);
          x[2 * b] = fmaf(lo, even.x, m);
          x[2 * b + 1] = fmaf(hi, odd.x, m);
          x[2 * b + 4] = fmaf(lo, even.y, m);
          x[2 * b + 5] = fmaf(hi, odd.y, m);
        }
        out[i * (D / 16)] = make_uint4(pack_value<T>(x[0], x[1]), pack_value<T>(x[2], x[3]), pack_value<T>(x[4], x[5]),
                                       pack_value<T>(x[6], x[7]));
      }
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads + 32, kBlocksPerSm) int4_gather_kernel(GatherParams p) {
  constexpr int kLanes = D / 16;
  constexpr int kGroups = kThreads / kLanes;
  // where a token's rows come from: >= 0: byte of its record, of head 0; -1: NaN; -2: nothing; <= -3: row -(src + 3) of
  // k_new / v_new.  And its row in the record.
  __shared__ long long s_src[2][kTokens];
  __shared__ int s_row[2][kTokens];
  const long long head_bytes = (long long)(p.page_size / kInt4Tokens) * int4_record_bytes(D);
  const int first_row = p.cu[0], end = min(p.total, p.cu[p.batch]);   // `total` may be an upper bound: the host never reads the lengths
  auto find = [&](int g0, int buf) {
    const int i = threadIdx.x - kThreads, g = g0 + i;
    if (i >= kTokens) return;
    long long src = -2;
    int row = 0;
    if (g >= first_row && g < end) {
      int lo = 0, hi = p.batch - 1;       // largest b with cu[b] <= g
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.cu[mid] <= g) lo = mid; else hi = mid - 1;
      }
      const int t = g - p.cu[lo];
      const int cached = p.cached ? p.cached[lo] : 0x7fffffff;
      if (cached < 0) {
        src = -1;                           // no such length: NaN
      } else if (p.cached && t >= cached) {
        const long long from = (long long)p.cu_new[lo] + t - cached;
        src = from >= 0 && from < p.cu_new[p.batch] ? -3 - from : -1;     // a row that k_new does not have reads as NaN
      } else {
        const int column = t / p.page_size, off = t - column * p.page_size;
        const int page = column < p.table_width ? p.table[int64_t(lo) * p.table_stride + column] : -1;
        src = page >= 0 && page < p.pool_pages      // a page outside the pool reads as NaN
                  ? (long long)page * p.heads_kv * head_bytes + (long long)(off / kInt4Tokens) * int4_record_bytes(D)
                  : -1;
        row = off % kInt4Tokens;
      }
    }
    s_src[buf][i] = src;
    s_row[buf][i] = row;
  };
  const bool finder = threadIdx.x >= kThreads;
  if (finder) find(blockIdx.x * kTokens, 0);
  __syncthreads();
  int buf = 0;
  for (int piece = blockIdx.x; piece * kTokens < end; piece += gridDim.x, buf ^= 1) {
    if (finder) {
      if ((piece + gridDim.x) * kTokens < end) find((piece + gridDim.x) * kTokens, buf ^ 1);
    } else {
      expand<T, D>(p, piece * kTokens, s_src[buf], s_row[buf], head_bytes);
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" int tb200_int4_cache_gather(const void* kv_pages, const int32_t* block_table, int64_t block_table_stride,
                                       int block_table_width, const int32_t* cu_seqlens_kv, const int32_t* cache_seqlens,
                                       const int32_t* cu_seqlens_new, const void* k_new, const void* v_new, void* k_out,
                                       void* v_out, int dtype, int total_tokens, int batch, int heads_kv, int dim,
                                       int page_size, int64_t pool_pages, void* stream) {
  if (total_tokens < 0 || batch <= 0 || heads_kv <= 0 || block_table_width <= 0)
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "batch, heads_kv and the table's width must be positive and total_tokens not negative");
  if (dtype != TB200_BF16 && dtype != TB200_F16) TB200_FAIL(TB200_ERR_UNSUPPORTED, "dtype must be F16 or BF16");
  if (dim != 64 && dim != 128) TB200_FAIL(TB200_ERR_UNSUPPORTED, "a 4-bit cache serves head dim 64 and 128, got %d", dim);
  if (page_size <= 0 || page_size % kInt4Tokens != 0)
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "page_size must be a multiple of 16, got %d", page_size);
  if (pool_pages < 0 || pool_pages > 0x7fffffffLL) TB200_FAIL(TB200_ERR_UNSUPPORTED, "too many pages");
  if (total_tokens > 1 << 30) TB200_FAIL(TB200_ERR_UNSUPPORTED, "at most 2^30 tokens");    // rows are counted in 32 bits
  if (total_tokens == 0) return TB200_OK;
  if (!kv_pages || !block_table || !cu_seqlens_kv || !k_out || !v_out)
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "kv_pages, block_table, cu_seqlens_kv, k_out and v_out must be non-null");
  if (cache_seqlens && (!cu_seqlens_new || !k_new || !v_new))
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "cache_seqlens comes with cu_seqlens_new, k_new and v_new");
  if ((reinterpret_cast<uintptr_t>(kv_pages) | reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out) |
       reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new)) & 15)
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "tensors must start on 16-byte boundaries");
  GatherParams p{};
  p.pages = static_cast<const unsigned char*>(kv_pages);
  p.table = block_table; p.table_stride = block_table_stride; p.table_width = block_table_width;
  p.cu = cu_seqlens_kv; p.cached = cache_seqlens; p.cu_new = cu_seqlens_new; p.k_new = k_new; p.v_new = v_new;
  p.k_out = k_out; p.v_out = v_out; p.batch = batch; p.heads_kv = heads_kv; p.page_size = page_size;
  p.pool_pages = int(pool_pages); p.total = total_tokens;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = dtype == TB200_BF16;
  const int pieces = (total_tokens + kTokens - 1) / kTokens, most = sm_count() * kBlocksPerSm;
  const int blocks = pieces < most ? pieces : most;
  if (dim == 64) {
    if (bf16) int4_gather_kernel<__nv_bfloat16, 64><<<blocks, kThreads + 32, 0, s>>>(p);
    else int4_gather_kernel<__half, 64><<<blocks, kThreads + 32, 0, s>>>(p);
  } else {
    if (bf16) int4_gather_kernel<__nv_bfloat16, 128><<<blocks, kThreads + 32, 0, s>>>(p);
    else int4_gather_kernel<__half, 128><<<blocks, kThreads + 32, 0, s>>>(p);
  }
  TB200_CUDA_CHECK(cudaGetLastError());
  return TB200_OK;
}
