// Block tables and slot maps of a paged KV cache, built on the GPU from the requests' lengths, sm_100a.
//
// A step appends new_lens[b] tokens to request b, which holds seq_lens[b].  With P = page_size
//   held_b = ceil(seq_b / P),  need_b = ceil((seq_b + new_b) / P) - held_b
//   C_b    = need_0 + .. + need_b          (requests whose lengths make no sense count as 0)
//   granted_b = sensible and (need_b == 0 or C_b <= free_count)
// The j-th new page of a granted request is free_pages[free_count - 1 - (C_b - need_b) - j]: pages come off the top of
// the stack in the order of the requests, and since C_b never falls, the pages that granted requests take are exactly
// the top of the stack.  Row t of the packed batch (request b, its i-th new token) sits at position seq_b + i and slot
// table[b][position / P] * P + position % P.
//
// Without a stack (free_count NULL) the table is taken to hold every page already, and only the maps are built.
//
// Latency bound: a few KB in and out.  One cluster of 1 to 8 blocks, one launch: every block scans all requests (it
// needs the offsets anyway), the cluster meets once, and then writes; so seq_lens and free_count may be updated in
// place without a second launch or a counter in memory.  Rows of the slot map go four to a thread (one binary search
// and two 16-byte stores per four rows); positions of new pages are computed from the stack, not read back from the table.
#include <cooperative_groups.h>

#include "tb200_common.cuh"

namespace tb200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kPlanThreads = 1024;
constexpr int kMaxRequests = 4096;
constexpr int kPerThread = kMaxRequests / kPlanThreads;
constexpr int kWarps = kPlanThreads / 32;

struct PlanParams {
  const int32_t* seq_lens;
  const int32_t* new_lens;
  int32_t* table;
  int64_t table_stride;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t *cu, *slots, *positions, *seq_after, *free_after, *granted;
  int batch, width, page, total, capacity;
};

struct PlanShared {
  int seq[kMaxRequests];
  int cu[kMaxRequests + 1];
  int taken[kMaxRequests];    // C_b - need_b: pages that the requests in front take
  int need[kMaxRequests];     // -1: not granted
  long long sums[2][kWarps];
  int last;
};

// Exclusive scan of one value per thread over the block, in 64 bits; *total gets the sum.
__device__ __forceinline__ long long block_scan(long long v, long long* sums, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  long long base = 0, all = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) base += sums[w];
    all += sums[w];
  }
  *total = all;
  return base + incl - v;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PlanParams p) {
  extern __shared__ unsigned char smem[];
  PlanShared& s = *reinterpret_cast<PlanShared*>(smem);
  const int tid = threadIdx.x;
  const int rank = int(blockIdx.x), blocks = int(gridDim.x);   // the grid is one cluster
  const bool allocates = p.free_count != nullptr;   // else the table holds every page already
  const int free_count = allocates ? min(max(*p.free_count, 0), p.capacity) : 0;
  const long long room = (long long)p.width * p.page;

  // requests tid * kPerThread ..
  int seq[kPerThread], fresh[kPerThread], need[kPerThread];
  bool fits[kPerThread];
  long long my_new = 0, my_need = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * kPerThread + i;
    seq[i] = 0; fresh[i] = 0; need[i] = 0; fits[i] = false;
    if (b < p.batch) {
      seq[i] = p.seq_lens[b];
      fresh[i] = p.new_lens[b];
      fits[i] = seq[i] >= 0 && fresh[i] >= 0 && (long long)seq[i] + fresh[i] <= room;
      if (fits[i] && allocates)
        need[i] = int(((long long)seq[i] + fresh[i] + p.page - 1) / p.page - ((long long)seq[i] + p.page - 1) / p.page);
      fresh[i] = max(fresh[i], 0);
    }
    my_new += fresh[i];
    my_need += need[i];
  }
  long long all_new, all_need;
  long long row = block_scan(my_new, s.sums[0], &all_new);
  long long taken = block_scan(my_need, s.sums[1], &all_need);
  if (tid == 0) s.last = 0;
  __syncthreads();
  long long most = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * kPerThread + i;
    if (b < p.batch) {
      const bool granted = fits[i] && (need[i] == 0 || taken + need[i] <= free_count);
      s.seq[b] = seq[i];
      s.cu[b] = int(min(row, 0x7fffffffLL));
      s.taken[b] = int(min(taken, 0x7fffffffLL));
      s.need[b] = granted ? need[i] : -1;
      if (granted && need[i] > 0) most = taken + need[i];
    }
    row += fresh[i];
    taken += need[i];
  }
  if (most > 0) atomicMax(&s.last, int(most));
  if (tid == 0) s.cu[p.batch] = int(min(all_new, 0x7fffffffLL));
  // every block has read the lengths and the count before any block writes them
  cg::this_cluster().sync();

  const int gtid = rank * kPlanThreads + tid, gthreads = blocks * kPlanThreads;
  for (int b = gtid; b <= p.batch; b += gthreads) {
    p.cu[b] = s.cu[b];
    if (b == p.batch) continue;
    const bool granted = s.need[b] >= 0;
    p.granted[b] = granted ? 1 : 0;
    p.seq_after[b] = granted ? s.seq[b] + (s.cu[b + 1] - s.cu[b]) : s.seq[b];
  }
  if (gtid == 0 && p.free_after) *p.free_after = free_count - s.last;

  // new entries of the table: a warp per request
  const int lane = tid & 31;
  for (int b = gtid >> 5; b < p.batch; b += gthreads >> 5) {
    const int n = s.need[b];
    if (n <= 0) continue;
    const int held = (s.seq[b] + p.page - 1) / p.page;
    for (int j = lane; j < n; j += 32)
      p.table[b * p.table_stride + held + j] = p.free_pages[free_count - 1 - s.taken[b] - j];
  }

  // slots and positions: four rows per thread
  for (int t0 = gtid * 4; t0 < p.total; t0 += gthreads * 4) {
    int slot[4], pos[4];
    int lo = 0, hi = p.batch - 1;    // largest b with cu[b] <= t0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s.cu[mid] <= t0) lo = mid; else hi = mid - 1;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = t0 + e;
      while (lo < p.batch - 1 && s.cu[lo + 1] <= t) ++lo;   // also steps over requests without a new token
      slot[e] = -1;
      pos[e] = 0;
      if (t < s.cu[p.batch]) {
        pos[e] = s.seq[lo] + (t - s.cu[lo]);
        if (s.need[lo] >= 0) {
          const int held = allocates ? (s.seq[lo] + p.page - 1) / p.page : p.width, column = pos[e] / p.page;
          const int id = column < held ? p.table[lo * p.table_stride + column]
                                       : p.free_pages[free_count - 1 - s.taken[lo] - (column - held)];
          slot[e] = id * p.page + (pos[e] - column * p.page);
        }
      }
    }
    if (t0 + 4 <= p.total && ((reinterpret_cast<uintptr_t>(p.slots) | reinterpret_cast<uintptr_t>(p.positions)) & 15) == 0) {
      *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (t0 + e < p.total) {
          p.slots[t0 + e] = slot[e];
          p.positions[t0 + e] = pos[e];
        }
      }
    }
  }
}

// Pages of the finished requests go back on the stack, request after request, a request's last page first (so that its
// first page is the next one handed out).  One block: reads and writes of the lengths are ordered by its barriers.
__global__ void __launch_bounds__(kPlanThreads) paged_release_kernel(const uint8_t* finished, int32_t* seq_lens,
                                                                     const int32_t* table, int64_t table_stride,
                                                                     int32_t* free_pages, int32_t* free_count, int capacity,
                                                                     int batch, int width, int page) {
  extern __shared__ unsigned char smem[];
  PlanShared& s = *reinterpret_cast<PlanShared*>(smem);
  const int tid = threadIdx.x;
  const int count = min(max(*free_count, 0), capacity);
  int held[kPerThread];
  long long mine = 0, all;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * kPerThread + i;
    held[i] = 0;
    if (b < batch && finished[b])
      held[i] = int(min((long long)width, ((long long)max(seq_lens[b], 0) + page - 1) / page));
    mine += held[i];
  }
  long long at = block_scan(mine, s.sums[0], &all);
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * kPerThread + i;
    if (b < batch) {
      s.need[b] = held[i];
      s.taken[b] = int(min(at, 0x7fffffffLL));
      if (finished[b]) seq_lens[b] = 0;
    }
    at += held[i];
  }
  __syncthreads();
  const int lane = tid & 31;
  for (int b = tid >> 5; b < batch; b += kWarps) {
    for (int j = lane; j < s.need[b]; j += 32) {
      const long long dst = (long long)count + s.taken[b] + j;
      if (dst < capacity) free_pages[dst] = table[b * table_stride + (s.need[b] - 1 - j)];
    }
  }
  if (tid == 0) *free_count = int(min((long long)capacity, count + all));
}

template <typename K>
int raise_shared_memory(K kern) {
  static thread_local bool done[64] = {false};
  int dev = 0;
  TB200_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) TB200_FAIL(TB200_ERR_UNSUPPORTED, "device index %d", dev);
  if (!done[dev]) {
    TB200_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(PlanShared))));
    done[dev] = true;
  }
  return TB200_OK;
}

int check_plan_sizes(int batch, int width, int page, int64_t capacity) {
  if (batch <= 0 || width <= 0 || page <= 0) TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "batch, pages per request and page_size must be positive");
  if (batch > kMaxRequests) TB200_FAIL(TB200_ERR_UNSUPPORTED, "at most %d requests, got %d", kMaxRequests, batch);
  if ((long long)width * page > 0x40000000LL) TB200_FAIL(TB200_ERR_UNSUPPORTED, "a request must hold at most 2^30 tokens");
  if (capacity < 0 || capacity > 0x7fffffffLL) TB200_FAIL(TB200_ERR_UNSUPPORTED, "too many pages");
  return TB200_OK;
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" int tb200_paged_kv_plan(const int32_t* seq_lens, const int32_t* new_lens, int32_t* block_table,
                                   int64_t block_table_stride, const int32_t* free_pages, int64_t free_capacity,
                                   const int32_t* free_count, int32_t* cu_seqlens, int32_t* slots, int32_t* positions,
                                   int32_t* seq_lens_after, int32_t* free_count_after, int32_t* granted, int batch,
                                   int max_pages_per_req, int page_size, int total_tokens, void* stream) {
  if (const int st = check_plan_sizes(batch, max_pages_per_req, page_size, free_capacity)) return st;
  if (total_tokens < 0) TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "total_tokens must not be negative");
  if (!seq_lens || !new_lens || !block_table || !cu_seqlens || !seq_lens_after || !granted ||
      (free_count && (!free_count_after || (free_capacity > 0 && !free_pages))) ||
      (total_tokens > 0 && (!slots || !positions)))
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "pointers must be non-null");
  if (const int st = raise_shared_memory(paged_plan_kernel)) return st;
  PlanParams p{seq_lens, new_lens, block_table, block_table_stride, free_pages, free_count, cu_seqlens, slots, positions,
               seq_lens_after, free_count_after, granted, batch, max_pages_per_req, page_size, total_tokens,
               int(free_capacity)};
  // one block covers 4096 rows per sweep
  const int blocks = total_tokens <= 4 * kPlanThreads ? 1 : total_tokens <= 8 * kPlanThreads ? 2
                   : total_tokens <= 16 * kPlanThreads ? 4 : 8;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = sizeof(PlanShared);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TB200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_plan_kernel, p));
  return TB200_OK;
}

extern "C" int tb200_paged_kv_release(const uint8_t* finished, int32_t* seq_lens, const int32_t* block_table,
                                      int64_t block_table_stride, int32_t* free_pages, int64_t free_capacity,
                                      int32_t* free_count, int batch, int max_pages_per_req, int page_size, void* stream) {
  if (const int st = check_plan_sizes(batch, max_pages_per_req, page_size, free_capacity)) return st;
  if (!finished || !seq_lens || !block_table || !free_count || (free_capacity > 0 && !free_pages))
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "pointers must be non-null");
  if (const int st = raise_shared_memory(paged_release_kernel)) return st;
  paged_release_kernel<<<1, kPlanThreads, sizeof(PlanShared), static_cast<cudaStream_t>(stream)>>>(
      finished, seq_lens, block_table, block_table_stride, free_pages, free_count, int(free_capacity), batch,
      max_pages_per_req, page_size);
  TB200_CUDA_CHECK(cudaGetLastError());
  return TB200_OK;
}
