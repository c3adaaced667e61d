// Single-token GQA decode over a paged cache held in 4 bits, sm_100a.
//
// Per q head, with the cached values k = ks * c + km and v = vs * c + vm (codes c = 0..15):
//   score_t = sm_scale * (ks_t * (q . c_t) + km_t * sum(q)),   softcap and mask, p_t = exp(score_t - max)
//   o = (sum_t p_t vs_t c_t + sum_t p_t vm_t) / sum_t p_t
//
// One block per (sequence, KV head, block of q heads); each of its warps takes every fourth token.
#include "int4_cache.cuh"

namespace tb200 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kHeadsPerBlock = 8;

struct Int4DecodeParams {
  const void* q;
  const unsigned char* pages;
  void* o;
  float* lse;
  const int32_t* lens;
  const int32_t* table;
  int64_t table_stride;
  int table_width, pool_pages, heads, heads_kv, group, page_size;
  float sm_scale, softcap;
};

template <typename T, typename TO, int D>
__global__ void __launch_bounds__(kThreads) gqa_decode_int4_kernel(Int4DecodeParams p) {
  constexpr int kDims = D / 32;    // dims of a lane
  __shared__ float s_o[kWarps][kHeadsPerBlock][D];
  __shared__ float s_m[kWarps][kHeadsPerBlock], s_l[kWarps][kHeadsPerBlock];
  const int b = blockIdx.x / p.heads_kv, hk = blockIdx.x % p.heads_kv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = blockIdx.y * kHeadsPerBlock;
  const int n_heads = min(kHeadsPerBlock, p.group - first);
  const int head0 = hk * p.group + first;
  const int capacity = int(min((long long)p.table_width * p.page_size, 0x7fffffffLL));
  int len = max(p.lens[b], 0);
  const bool too_long = len > capacity;
  if (too_long) len = capacity;
  float q[kHeadsPerBlock][kDims], o[kHeadsPerBlock][kDims], m[kHeadsPerBlock], l[kHeadsPerBlock];
#pragma unroll
  for (int h = 0; h < kHeadsPerBlock; ++h) {
    m[h] = kNegFloor;
    l[h] = 0.f;
#pragma unroll
    for (int e = 0; e < kDims; ++e) {
      o[h][e] = 0.f;
      q[h][e] = h < n_heads ? float(static_cast<const T*>(p.q)[(size_t(b) * p.heads + head0 + h) * D + lane * kDims + e]) : 0.f;
    }
  }
  for (int t = warp; t < len; t += kWarps) {
    const int page = p.table[b * p.table_stride + t / p.page_size];
    const bool known = !too_long && page >= 0 && page < p.pool_pages;
    float k[kDims], v[kDims];
#pragma unroll
    for (int e = 0; e < kDims; ++e) k[e] = v[e] = __int_as_float(0x7fc00000);
    if (known) {
      const int off = t % p.page_size, tok = off % kInt4Tokens;
      const unsigned char* rec =
          p.pages + ((size_t(page) * p.heads_kv + hk) * size_t(p.page_size / kInt4Tokens) + off / kInt4Tokens) *
                        size_t(int4_record_bytes(D));
      const __half* params = reinterpret_cast<const __half*>(rec + kInt4Tokens * D + tok * 8);
      const float ks = __half2float(params[0]), km = __half2float(params[1]);
      const float vs = __half2float(params[2]), vm = __half2float(params[3]);
#pragma unroll
      for (int e = 0; e < kDims; e += 2) {
        const unsigned kb = rec[tok * (D / 2) + (lane * kDims + e) / 2];
        const unsigned vb = rec[(kInt4Tokens + tok) * (D / 2) + (lane * kDims + e) / 2];
        k[e] = fmaf(ks, float(kb & 15u), km);
        k[e + 1] = fmaf(ks, float(kb >> 4), km);
        v[e] = fmaf(vs, float(vb & 15u), vm);
        v[e + 1] = fmaf(vs, float(vb >> 4), vm);
      }
    }
#pragma unroll
    for (int h = 0; h < kHeadsPerBlock; ++h) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < kDims; ++e) s = fmaf(q[h][e], k[e], s);
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= p.sm_scale;
      if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
      s *= kLog2e;
      const float mn = s != s || m[h] != m[h] ? NAN : fmaxf(m[h], s);
      const float a = exp2f(m[h] - mn), w = exp2f(s - mn);
      m[h] = mn;
      l[h] = l[h] * a + w;
#pragma unroll
      for (int e = 0; e < kDims; ++e) o[h][e] = o[h][e] * a + w * v[e];
    }
  }
#pragma unroll
  for (int h = 0; h < kHeadsPerBlock; ++h) {
#pragma unroll
    for (int e = 0; e < kDims; ++e) s_o[warp][h][lane * kDims + e] = o[h][e];
    if (lane == 0) {
      s_m[warp][h] = m[h];
      s_l[warp][h] = l[h];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_heads * D; i += kThreads) {
    const int h = i / D, d = i - h * D;
    float M = kNegFloor, L = 0.f, acc = 0.f;
    for (int w = 0; w < kWarps; ++w) M = M != M || s_m[w][h] != s_m[w][h] ? NAN : fmaxf(M, s_m[w][h]);
    for (int w = 0; w < kWarps; ++w) {
      const float a = exp2f(s_m[w][h] - M);
      L += a * s_l[w][h];
      acc += a * s_o[w][h][d];
    }
    const size_t row = size_t(b) * p.heads + head0 + h;
    const bool empty = L == 0.f;
    store_out<TO>(static_cast<TO*>(p.o) + row * D + d, empty ? 0.f : acc / L);
    if (d == 0 && p.lse) p.lse[row] = empty ? -INFINITY : M + log2f(L);
  }
}

template <typename T, int D>
void launch_o(const Int4DecodeParams& p, int batch, int o_dtype, cudaStream_t s) {
  const dim3 grid(batch * p.heads_kv, (p.group + kHeadsPerBlock - 1) / kHeadsPerBlock);
  if (o_dtype == TB200_F32) gqa_decode_int4_kernel<T, float, D><<<grid, kThreads, 0, s>>>(p);
  else if (o_dtype == TB200_BF16) gqa_decode_int4_kernel<T, __nv_bfloat16, D><<<grid, kThreads, 0, s>>>(p);
  else gqa_decode_int4_kernel<T, __half, D><<<grid, kThreads, 0, s>>>(p);
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" size_t tb200_gqa_decode_int4_workspace_bytes(int batch, int heads, int heads_kv, int dim) {
  if (batch <= 0 || heads <= 0 || heads_kv <= 0 || heads % heads_kv != 0 || (dim != 64 && dim != 128)) return 0;
  return 256;
}

extern "C" int tb200_gqa_decode_int4(const void* q, const void* kv_pages, void* o, float* lse,
                                     const int32_t* real_seqlen_kv, const int32_t* block_table,
                                     int64_t block_table_stride, int block_table_width, int q_dtype, int o_dtype,
                                     int batch, int heads, int heads_kv, int dim, int page_size, int64_t pool_pages,
                                     float sm_scale, float softcap, int flags, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  if (!q || !kv_pages || !o || !real_seqlen_kv || !block_table || !workspace)
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "q, kv_pages, o, real_seqlen_kv, block_table and workspace must be non-null");
  if (batch <= 0 || heads <= 0 || heads_kv <= 0 || block_table_width <= 0 || block_table_stride < 0)
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "batch, heads, heads_kv and the table's width must be positive");
  if (heads % heads_kv != 0) TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "heads must be divisible by heads_kv");
  if (dim != 64 && dim != 128) TB200_FAIL(TB200_ERR_UNSUPPORTED, "a 4-bit cache serves head dim 64 and 128, got %d", dim);
  if (page_size <= 0 || page_size % kInt4Tokens != 0)
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "page_size must be a multiple of 16, got %d", page_size);
  if (q_dtype != TB200_BF16 && q_dtype != TB200_F16) TB200_FAIL(TB200_ERR_UNSUPPORTED, "q must be F16 or BF16");
  if (o_dtype != TB200_F32 && o_dtype != TB200_BF16 && o_dtype != TB200_F16)
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "o must be F16, BF16 or F32");
  if (pool_pages <= 0 || pool_pages > 0x7fffffffLL) TB200_FAIL(TB200_ERR_UNSUPPORTED, "the pool must hold 1 to 2^31 - 1 pages");
  Int4DecodeParams p{};
  p.q = q; p.pages = static_cast<const unsigned char*>(kv_pages); p.o = o; p.lse = lse; p.lens = real_seqlen_kv;
  p.table = block_table; p.table_stride = block_table_stride; p.table_width = block_table_width;
  p.pool_pages = int(pool_pages); p.heads = heads; p.heads_kv = heads_kv; p.group = heads / heads_kv;
  p.page_size = page_size; p.sm_scale = sm_scale; p.softcap = softcap;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (q_dtype == TB200_BF16) {
    if (dim == 64) launch_o<__nv_bfloat16, 64>(p, batch, o_dtype, s);
    else launch_o<__nv_bfloat16, 128>(p, batch, o_dtype, s);
  } else {
    if (dim == 64) launch_o<__half, 64>(p, batch, o_dtype, s);
    else launch_o<__half, 128>(p, batch, o_dtype, s);
  }
  TB200_CUDA_CHECK(cudaGetLastError());
  return TB200_OK;
}
