// Block tables and slot maps of a paged KV cache, built on the GPU from the requests' lengths, sm_100a.
//
// A step appends new_lens[b] tokens to request b, which holds seq_lens[b].  With P = page_size
//   held_b = ceil(seq_b / P),  need_b = ceil((seq_b + new_b) / P) - held_b
//   C_b    = need_0 + .. + need_b          (requests whose lengths make no sense count as 0)
//   granted_b = sensible and (need_b == 0 or C_b <= free_count)
// The j-th new page of a granted request is free_pages[free_count - 1 - (C_b - need_b) - j]: pages come off the top of
// the stack in the order of the requests, and since C_b never falls, the pages that granted requests take are exactly
// the top of the stack.  Row t of the packed batch (request b, its i-th new token) sits at position seq_b + i and slot
// table[b][position / P] * P + position % P, or -1 where the page id is negative or the slot does not fit 32 bits.
//
// Without a stack (free_count NULL) the table is taken to hold every page already, and only the maps are built.
//
// Latency bound: a few KB in and out, one launch.  Every block scans all requests (it needs the offsets anyway) and then
// writes its share.  Where seq_lens or free_count are updated in place the launch is one cluster of up to 8 blocks, which
// meets between reading and writing; else blocks need not know of each other.  Small steps run in small blocks (the scans'
// barriers cost more than the work: 64 requests take 9 us in a block of 1024 threads with serial sums over 32 warps, 5.4 as
// it is; 512 requests with 49.5 thousand rows 6.8; in place, where that is one cluster of eight blocks, 5.1
// and 12.4, beside 4.8 and 6.3 in the same program).
// Positions of new pages are computed from the stack, not read back from the table.
#include <cooperative_groups.h>

#include "tb200_common.cuh"

namespace tb200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kPlanThreads = 1024;     // at most
constexpr int kMaxRequests = 4096;
constexpr int kPerThread = 4;          // requests of a thread, at most

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

// Shared memory: four words per request, sized by the batch.
struct PlanShared {
  int* seq;
  int* cu;       // [batch + 1]
  int* taken;    // C_b - need_b: pages that the requests in front take
  int* need;     // -1: not granted
  __device__ __forceinline__ PlanShared(int* at, int batch)
      : seq(at), cu(at + batch), taken(at + 2 * batch + 1), need(at + 3 * batch + 1) {}
};
size_t plan_smem(int batch) { return (size_t(4) * batch + 1) * sizeof(int); }

// Exclusive scan of one value per thread over the block, in 64 bits; *total gets the sum.  `sums`: 32 words of its own.
__device__ __forceinline__ long long block_scan(long long v, long long* sums, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  const long long mine = lane < warps ? sums[lane] : 0;
  long long upto = mine;      // every warp scans the warps' sums
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += n;
  }
  *total = __shfl_sync(0xffffffffu, upto, 31);
  return __shfl_sync(0xffffffffu, upto - mine, warp) + incl - v;
}

// Largest b with cu[b] <= t.
__device__ __forceinline__ int find_request(const PlanShared& s, int batch, int t) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}
// Slot and position of row t, whose request is `lo` or one behind it (also steps over requests without a new token).
__device__ __forceinline__ void map_row(const PlanParams& p, const PlanShared& s, int t, int& lo, bool allocates, int free_count,
                                        int& slot, int& pos) {
  while (lo < p.batch - 1 && s.cu[lo + 1] <= t) ++lo;
  slot = -1;
  pos = 0;
  if (t >= s.cu[p.batch]) return;
  pos = s.seq[lo] + (t - s.cu[lo]);
  if (s.need[lo] < 0) return;
  const int held = allocates ? (s.seq[lo] + p.page - 1) / p.page : p.width, column = pos / p.page;
  const int id = column < held ? p.table[lo * p.table_stride + column]
                               : p.free_pages[free_count - 1 - s.taken[lo] - (column - held)];
  // In 64 bits: a page id that no pool has must not become a row of another page by wrapping.
  const long long at = (long long)id * p.page + (pos - column * p.page);
  if (id >= 0 && at <= 0x7fffffffLL) slot = int(at);
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PlanParams p) {
  extern __shared__ int smem[];
  __shared__ long long s_sums[2][32];
  __shared__ int s_last;
  const PlanShared s(smem, p.batch);
  const int tid = threadIdx.x, threads = blockDim.x;
  const int rank = int(blockIdx.x), blocks = int(gridDim.x);
  const int per = (p.batch + threads - 1) / threads;           // requests tid * per ..
  const bool allocates = p.free_count != nullptr;   // else the table holds every page already
  const int free_count = allocates ? min(max(*p.free_count, 0), p.capacity) : 0;
  const long long room = (long long)p.width * p.page;

  int seq[kPerThread], fresh[kPerThread], need[kPerThread];
  bool fits[kPerThread];
  long long my_new = 0, my_need = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * per + i;
    seq[i] = 0; fresh[i] = 0; need[i] = 0; fits[i] = false;
    if (i < per && b < p.batch) {
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
  long long row = block_scan(my_new, s_sums[0], &all_new);
  long long taken = block_scan(my_need, s_sums[1], &all_need);
  if (tid == 0) s_last = 0;
  __syncthreads();
  long long most = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * per + i;
    if (i < per && b < p.batch) {
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
  if (most > 0) atomicMax(&s_last, int(most));
  if (tid == 0) s.cu[p.batch] = int(min(all_new, 0x7fffffffLL));
  // every block has read the lengths and the count before any block writes them
  cg::this_cluster().sync();

  const int gtid = rank * threads + tid, gthreads = blocks * threads;
  for (int b = gtid; b <= p.batch; b += gthreads) {
    p.cu[b] = s.cu[b];
    if (b == p.batch) continue;
    const bool granted = s.need[b] >= 0;
    p.granted[b] = granted ? 1 : 0;
    p.seq_after[b] = granted ? s.seq[b] + (s.cu[b + 1] - s.cu[b]) : s.seq[b];
  }
  if (gtid == 0 && p.free_after) *p.free_after = free_count - s_last;

  // new entries of the table: a warp per request
  const int lane = tid & 31;
  for (int b = gtid >> 5; b < p.batch; b += gthreads >> 5) {
    const int n = s.need[b];
    if (n <= 0) continue;
    const int held = (s.seq[b] + p.page - 1) / p.page;
    for (int j = lane; j < n; j += 32)
      p.table[b * p.table_stride + held + j] = p.free_pages[free_count - 1 - s.taken[b] - j];
  }

  // slots and positions: a row per thread where that does, else four
  if (p.total <= gthreads) {
    if (gtid < p.total) {
      int slot, pos, request = find_request(s, p.batch, gtid);
      map_row(p, s, gtid, request, allocates, free_count, slot, pos);
      p.slots[gtid] = slot;
      p.positions[gtid] = pos;
    }
    return;
  }
  for (int t0 = gtid * 4; t0 < p.total; t0 += gthreads * 4) {
    int slot[4], pos[4], request = find_request(s, p.batch, t0);
#pragma unroll
    for (int e = 0; e < 4; ++e) map_row(p, s, t0 + e, request, allocates, free_count, slot[e], pos[e]);
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
  extern __shared__ int smem[];
  __shared__ long long s_sums[32];
  const PlanShared s(smem, batch);
  const int tid = threadIdx.x, threads = blockDim.x;
  const int per = (batch + threads - 1) / threads;
  const int count = min(max(*free_count, 0), capacity);
  int held[kPerThread];
  long long mine = 0, all;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * per + i;
    held[i] = 0;
    if (i < per && b < batch && finished[b])
      held[i] = int(min((long long)width, ((long long)max(seq_lens[b], 0) + page - 1) / page));
    mine += held[i];
  }
  long long at = block_scan(mine, s_sums, &all);
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = tid * per + i;
    if (i < per && b < batch) {
      s.need[b] = held[i];
      s.taken[b] = int(min(at, 0x7fffffffLL));
      if (finished[b]) seq_lens[b] = 0;
    }
    at += held[i];
  }
  __syncthreads();
  const int lane = tid & 31;
  for (int b = tid >> 5; b < batch; b += threads >> 5) {
    for (int j = lane; j < s.need[b]; j += 32) {
      const long long dst = (long long)count + s.taken[b] + j;
      if (dst < capacity) free_pages[dst] = table[b * table_stride + (s.need[b] - 1 - j)];
    }
  }
  if (tid == 0) *free_count = int(min((long long)capacity, count + all));
}

// Threads of a block: one for every request (four at most share a thread), and enough for the rows of a small step.
int plan_threads(int batch, int total) {
  const int want = batch > total ? batch : total;
  return want <= 128 ? 128 : want <= 256 ? 256 : want <= 512 ? 512 : kPlanThreads;
}

// More shared memory than a function has by itself.  The limit belongs to the function and not to this thread: every thread
// sets the one that the largest batch needs, so that none takes it from another between its own setting and its launch.
int allow_largest_batch(size_t smem) {
  if (smem <= 48 * 1024) return TB200_OK;
  const int most = int(plan_smem(kMaxRequests));
  TB200_CUDA_CHECK(cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  TB200_CUDA_CHECK(cudaFuncSetAttribute(paged_release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
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
  if (total_tokens > 1 << 30) TB200_FAIL(TB200_ERR_UNSUPPORTED, "at most 2^30 tokens");    // rows are counted in 32 bits
  if (!seq_lens || !new_lens || !block_table || !cu_seqlens || !seq_lens_after || !granted ||
      (free_count && (!free_count_after || (free_capacity > 0 && !free_pages))) ||
      (total_tokens > 0 && (!slots || !positions)))
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "pointers must be non-null");
  PlanParams p{seq_lens, new_lens, block_table, block_table_stride, free_pages, free_count, cu_seqlens, slots, positions,
               seq_lens_after, free_count_after, granted, batch, max_pages_per_req, page_size, total_tokens,
               int(free_capacity)};
  const int threads = plan_threads(batch, total_tokens);
  const bool in_place = seq_lens_after == seq_lens || (free_count && free_count_after == free_count);
  int blocks = (total_tokens + threads - 1) / threads;
  blocks = blocks < 1 ? 1 : blocks;
  if (in_place) {
    blocks = blocks > 4 ? 8 : blocks > 2 ? 4 : blocks;
  } else if (blocks > sm_count()) {
    blocks = sm_count();
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = plan_smem(batch);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = in_place ? blocks : 1;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (const int st = allow_largest_batch(cfg.dynamicSmemBytes)) return st;
  TB200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_plan_kernel, p));
  return TB200_OK;
}

extern "C" int tb200_paged_kv_release(const uint8_t* finished, int32_t* seq_lens, const int32_t* block_table,
                                      int64_t block_table_stride, int32_t* free_pages, int64_t free_capacity,
                                      int32_t* free_count, int batch, int max_pages_per_req, int page_size, void* stream) {
  if (const int st = check_plan_sizes(batch, max_pages_per_req, page_size, free_capacity)) return st;
  if (!finished || !seq_lens || !block_table || !free_count || (free_capacity > 0 && !free_pages))
    TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "pointers must be non-null");
  const size_t smem = plan_smem(batch);
  if (const int st = allow_largest_batch(smem)) return st;
  paged_release_kernel<<<1, plan_threads(batch, 0), smem, static_cast<cudaStream_t>(stream)>>>(
      finished, seq_lens, block_table, block_table_stride, free_pages, free_count, int(free_capacity), batch,
      max_pages_per_req, page_size);
  TB200_CUDA_CHECK(cudaGetLastError());
  return TB200_OK;
}
