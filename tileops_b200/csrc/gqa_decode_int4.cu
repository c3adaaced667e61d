// Single-token GQA decode over a paged cache held in 4 bits, sm_100a.
//
// Per q head, with the cached values k = ks * c + km and v = vs * c + vm (codes c = 0..15):
//   score_t = sm_scale * (ks_t * (q . c_t) + km_t * sum(q)),   softcap and mask, p_t = 2^(log2e score_t - max)
//   o = (sum_t (p_t vs_t) c_t + sum_t p_t vm_t) / sum_t p_t
// so the tensor cores see bare codes; scales and offsets meet them in fp32, once per (token, head).
//
// HBM bound: dim + 8 bytes per token and KV head.  The floor asks every SM for 16 tokens of one head per ~94 clocks, i.e.
// 2 * 16 * 128 codes expanded in 375 issue slots of its four schedulers, whose logic pipe takes an instruction every other
// clock: the expansion has to be cheap, and no code is converted.
//   K: a nibble masked into a byte is an operand of the integer MMA (m16n8k32, u8 x s8): one AND per four codes, 3 logic
//      instructions per 8 codes.  q becomes an integer of two signed bytes (bf16; 2^13 <= max |q| < 2^14 after a power of
//      two per head: exact for values above 2^-6 of the largest, else within 2^-14 of it) or three (fp16).
//   V: the product runs over tokens, so a register holds two tokens of one dim in float16: the nibble n0 masked into zeros
//      IS the subnormal n0 * 2^-24, which the tensor cores multiply exactly, and the byte n0 + 16 n1 as it stands is its
//      neighbour's operand, from which the epilogue subtracts the first row's sum: 5 logic instructions per 8 codes, the
//      gather of two tokens into a register included.
//   (With float16 nibbles for both, 5 and 6 instructions, the logic pipe was 57 % busy at half of the memory's rate: 70 us
//   for 8 x 32768 tokens of 8 heads x 128.  e4m3 operands, where 0..15 are numbers too, are converted by mma.sync itself:
//   24 clocks an MMA against 8.)
//
//   * Tokens on the MMA's M dimension, q heads on N = 8: at most 16 rows of q per KV head are too few for a tcgen05 tile,
//     and the matrix work is a small part of what the warp-level unit can do.
//   * P * vs is scaled by a running power of two above every |vs| seen and rounded to float16.  That rounding meets the
//     codes' distance from 7.5 only: sum p (vm + 7.5 vs) is added in fp32, and 7.5 * sum of the ROUNDED weights, one more
//     MMA against a constant, is taken off (error of an fp16 output 4.5e-4 without it).
//   * The running maximum moves only when a score exceeds it by 2^8: P * vs then stays below 2^15, sums are fp32, and the
//     rescaling of the accumulators, the shuffles of the maximum and their latency leave the inner loop.
//   * Rows of a record are dealt to the MMA rows in the order 0 7 1 6 2 5 3 4: the pairs a lane needs of V (consecutive k
//     of the second product) and the rows it reads of K then fall into different banks.
//   * At most four q heads per KV head leave half of N idle: the second digit of q takes it, the lanes of the two halves
//     exchange what the other needs and have one token's scores of a record each (64 sequences of 512 to 8192 tokens, 297 MB,
//     67.2 -> 63.5 us).
//   * Three blocks of four math warps per SM (head dim 64: four; two head tiles: two), each with a producer warp that streams records by untiled bulk copies (as many
//     tokens as a page and a tile have in common, 16 at least) into a ring of shared-memory stages, across segment boundaries.
//     (One block of twelve math warps, which share every stage and every segment, repeats a segment's beginning and end in
//     twelve warps instead of four: 157 against 126 us on 128 sequences of 4096 tokens, 8 KV heads.)
//   * Work is cut into equal contiguous ranges, one per block (stream-K), as in gqa_decode_tma.cu; to begin and end a segment
//     counts as two or three tiles (without that 78 us instead of 69 on 64 sequences of 512 to 8192 tokens, whose short lanes
//     made the blocks that got them late).  Partial results of a (sequence, KV head) that ranges share go to global memory
//     in accumulator order; the last block to finish merges them, at the end of its range.
// Measured, 32 q and 8 KV heads x 128, bf16, captured: 8 x 131072 tokens 186 us = 6.1 TB/s (205 to 217 us back to back, where
// the board's power limit takes the clock to 1.65 GHz); 64 sequences of 512 to 8192 tokens, 325 MB, 67 us = 4.9 TB/s: of that 6 us pass
// before the first tile, 5 after the last, and each segment's begin and end cost its block 3; 1 x 1000 tokens 11 us, latency.
#include <type_traits>

#include "int4_cache.cuh"
#include "tb200_async.cuh"

namespace tb200 {
namespace {

constexpr int kMathThreads = 128;
constexpr int kWarps = 4;
constexpr int kAllThreads = kMathThreads + 32;
constexpr int kMathBarrier = 1;
constexpr int kItemSlots = 2;
constexpr int kCounterWords = 4;     // [0], [1] spare, [2] status, [3] spare; tickets follow
constexpr int kMaxBatch = 4096;
constexpr int kSlotsPerSm = 12;      // partial results that the workspace holds: 2 per range, a range per resident block
constexpr float kGrow = 8.f;         // a score this much (log2) above the running maximum moves it
constexpr int kPBits = 7;            // P * vs is scaled to 2^kPBits: 2^(kGrow + kPBits) < 65504
constexpr uint32_t kMid = 0x47804780u;   // 7.5 twice in float16

struct Int4DecodeParams {
  const void* q;
  const unsigned char* pages;
  void* o;
  float* lse;
  const int32_t* lens;
  const int32_t* table;
  int64_t table_stride;
  int table_width, pool_pages, batch, heads, heads_kv, group, page_size;
  int hb, n_hb;            // q heads of a head block, head blocks of a KV head
  int capacity;            // tokens a row of the table can name
  int records_per_copy;    // 16-token records that one bulk copy fetches: 1, 2, 4, .. a whole tile's
  float sm_scale, softcap;
  int force_chunk, max_slots;
  int* counters;
  float4* part_o;          // [max_slots][NT * D / 16][32 lanes]: accumulator fragments
  float4* part_ml;         // [max_slots][NT][4]: max and sum of heads 2 t, 2 t + 1
  long long wait_cycles;
};

template <int D, int NT>
struct Cfg {
  static constexpr int kRec = int4_record_bytes(D);
  static constexpr int R = 2;                                                 // records of a math warp per tile
  static constexpr int kRecords = kWarps * R;
  static constexpr int kTile = kRecords * kInt4Tokens;                        // tokens per tile
  static constexpr int kStageBytes = kRecords * kRec;
  static constexpr int kStages = D == 128 ? 3 : 4;
  static constexpr int kBlocks = NT == 2 ? 2 : D == 128 ? 3 : 4;              // per SM
  static constexpr unsigned kMinRun = D == 128 ? 3 : 4;       // tiles of a run, at least
  static constexpr unsigned kSegmentCost = D == 128 ? 2 : 3;  // tiles' worth of time to begin and end a segment
  static constexpr int kHeads = 8 * NT;
  static constexpr int kQSlotBytes = kHeads * D * 2;
  static constexpr int kFrags = NT * D / 16;             // accumulator fragments of a warp
  static constexpr int ring = 0;
  static constexpr int qslots = ring + kStages * kStageBytes;
  static constexpr int dump = qslots + kItemSlots * kQSlotBytes;              // [kWarps][kFrags][32] float4
  static constexpr int ml = dump + kWarps * kFrags * 512;                     // [kWarps][NT][4] float4
  static constexpr int bars = ml + kWarps * NT * 64;
  static constexpr int segs = bars + 8 * (2 * kStages + 2 * kItemSlots + 2);  // [kItemSlots] Segment
  static constexpr int ends = segs + kItemSlots * 64;                         // Segments: the range's first, its last so far, the current
  static constexpr int misc = ends + 3 * 64;                                  // 20 ints
  static constexpr int plan = misc + 80;                                      // s_prefix [batch + 1], s_lens [batch]
  static_assert(kSegmentCost < kMinRun, "no range lies in a gap");
  static_assert(2 * kBlocks <= kSlotsPerSm, "every range has its slots");
  static_assert(qslots % 128 == 0 && dump % 16 == 0 && bars % 8 == 0, "layout");
  static_assert(plan + (2 * kMaxBatch + 1) * 4 <= 227 * 1024, "the largest batch fits a block");
};

template <int D, int NT>
size_t smem_bytes(int batch) {
  return size_t(Cfg<D, NT>::plan) + size_t(2 * batch + 1) * 4;
}

// A segment: the tiles of one lane (sequence, KV head, head block) that one range of the partition covers.
struct alignas(16) Segment {
  int b, hk, hbi, len;
  int tile0, tile1, n_runs, slot;
  unsigned lane_start, next;
  int first_range, lane;
  int too_long;
};
static_assert(sizeof(Segment) <= 64, "a slot of shared memory");
// Slot of the partial result that range k contributes to the lane that starts at unit lane_start.
__device__ __forceinline__ int segment_slot(int k, unsigned per, unsigned lane_start) {
  return 2 * k + (unsigned(k) * per >= lane_start ? 0 : 1);
}
// The segment at unit u of a range that ends at range_end.  Lanes lie `gap` units apart; `even` is their width where all
// sequences have the same number of tiles, else 0.
__device__ __forceinline__ Segment segment_at(const Int4DecodeParams& p, unsigned u, unsigned range_begin,
                                              unsigned range_end, int range, unsigned per, unsigned gap, unsigned even,
                                              const int* s_prefix, const int* s_lens) {
  Segment g;
  const int lanes = p.heads_kv * p.n_hb;
  int lo = 0;
  unsigned width = even, base;
  if (even) {
    lo = int(u / (even * unsigned(lanes)));
    base = unsigned(lo) * even * unsigned(lanes);
  } else {
    int hi = p.batch - 1;   // largest b with lanes * prefix[b] <= u
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (unsigned(s_prefix[mid]) * unsigned(lanes) <= u) lo = mid; else hi = mid - 1;
    }
    width = unsigned(s_prefix[lo + 1] - s_prefix[lo]);
    base = unsigned(s_prefix[lo]) * unsigned(lanes);
  }
  g.b = lo;
  const int len = max(s_lens[lo], 0);
  g.too_long = len > p.capacity;
  g.len = min(len, p.capacity);
  const int rem = int((u - base) / width);
  g.hk = p.n_hb == 1 ? rem : rem / p.n_hb;
  g.hbi = rem - g.hk * p.n_hb;
  g.lane = lo * lanes + rem;
  g.lane_start = base + unsigned(rem) * width + gap;
  const unsigned lane_end = g.lane_start + width - gap, begin = max(u, g.lane_start);
  g.tile0 = int(begin - g.lane_start);
  g.tile1 = int(min(range_end, lane_end) - g.lane_start);
  g.next = lane_end + gap < range_end ? lane_end : range_end;     // no tile lies in what the range holds of a gap
  const bool whole = g.lane_start >= range_begin && lane_end <= range_end;
  g.first_range = whole ? range : int(g.lane_start / per);
  g.n_runs = whole ? 1 : int((lane_end - 1) / per) - g.first_range + 1;
  g.slot = segment_slot(range, per, g.lane_start);
  return g;
}

// Units of the sequences: s_prefix[0..batch] = exclusive sums per lane, s_lens = lengths as given.  A lane has its tiles
// and, where lengths differ, kSegmentCost units in front of them for what it costs to begin and end one.  By the
// math threads.
template <int kTile, unsigned kSegmentCost>
__device__ __forceinline__ void tile_plan(const Int4DecodeParams& p, int tid, int* s_prefix, int* s_lens, int* s_sums,
                                          int* s_ragged) {
  const int lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + kMathThreads - 1) / kMathThreads;
  const int b0 = tid * per;
  const int first_tiles = (min(max(p.lens[0], 0), p.capacity) + kTile - 1) / kTile;
  int sum = 0, live = 0;
  bool ragged = false;
  for (int i = 0; i < per; ++i) {
    const int b = b0 + i;
    if (b < p.batch) {
      const int len = p.lens[b];
      s_lens[b] = len;
      const int t = (min(max(len, 0), p.capacity) + kTile - 1) / kTile;
      ragged |= t != first_tiles;
      sum += t;
      live += t > 0;
    }
  }
  ragged = __any_sync(0xffffffffu, ragged);
  int incl = sum, incl_live = live;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, incl, o), m = __shfl_up_sync(0xffffffffu, incl_live, o);
    if (lane >= o) { incl += n; incl_live += m; }
  }
  if (lane == 31) {
    s_sums[warp] = incl;
    s_sums[kWarps + warp] = incl_live;
    s_ragged[warp] = ragged ? 1 : 0;
  }
  named_barrier(kMathBarrier, kMathThreads);
  const int gap = (s_ragged[0] | s_ragged[1] | s_ragged[2] | s_ragged[3]) ? int(kSegmentCost) : 0;   // else added later
  int run = incl - sum + gap * (incl_live - live);
  for (int w = 0; w < warp; ++w) run += s_sums[w] + gap * s_sums[kWarps + w];
  for (int i = 0; i < per; ++i) {
    const int b = b0 + i;
    if (b < p.batch) {
      s_prefix[b] = run;
      const int t = (min(max(s_lens[b], 0), p.capacity) + kTile - 1) / kTile;
      run += t > 0 ? t + gap : 0;
    }
    if (b == p.batch - 1) s_prefix[p.batch] = run;
  }
}

// cap * tanh(x / cap) with tanh y = 1 - 2 / (1 + e^2y): off by a few 2^-24 of cap
__device__ __forceinline__ float soft_cap(float x, float cap, float inv_cap) {
  const float e = fast_exp2(x * inv_cap * (2.f * kLog2e));   // overflows to infinity, where the quotient is 0
  return cap - __fdividef(2.f * cap, 1.f + e);
}

__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127

// D(16x8, s32) = A(16x32, u8) * B(32x8, s8) + C, where C is D or (first) zero
__device__ __forceinline__ void mma_16832_u8s8(int (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], bool first) {
  if (first)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "r"(0));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// Code of the first wait on this device that ran out since the word was last cleared.  The workspace has one too, but that of a
// captured launch is a temporary of the graph, which clears it on every replay: this one stays until the host reads it.
__device__ int g_gave_up;

// As mbar_wait_bounded, with the first poll in line.
__device__ __forceinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code,
                                            long long limit, unsigned sleep) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (sleep) __nanosleep(sleep);     // a polling warp takes issue slots from the warps it waits for
    if (*abort_flag) return false;
    if (clock64() - t0 > limit) {
      *abort_flag = 1;
      atomicCAS(status, 0, code);
      atomicCAS(&g_gave_up, 0, code);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code,
                                          long long limit, unsigned sleep = 0) {
  if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_slow(bar, parity, abort_flag, status, code, limit, sleep);
}
// The same by a whole warp, whose lanes get one answer: where one of them gives up, none goes on to a shuffle or a vote that
// it no longer takes part in.  (64 ragged requests, 297 MB, 62.0 -> 62.5 us; 8 x 131072 tokens 184.9 -> 187.0 us.)
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code,
                                               long long limit) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait_slow(bar, parity, abort_flag, status, code, limit, 0));
}

template <int kWords>
__device__ __forceinline__ void lds_words(uint32_t (&w)[kWords], const unsigned char* at) {
  if constexpr (kWords == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(at);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else if constexpr (kWords == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(at);
    w[0] = u.x; w[1] = u.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(at);
  }
}

// Largest |x| of 2 N 16-bit values, of which NaN counts for nothing.
template <typename T, int N>
__device__ __forceinline__ float abs_max(const uint32_t (&x)[N]) {
  if constexpr (std::is_same<T, __half>::value) {
    __half2 m = __float2half2_rn(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&x[i])));
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    __nv_bfloat162 m = __float2bfloat162_rn(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&x[i])));
    return fmaxf(__low2float(m), __high2float(m));
  }
}

// A sum of partial results (fragments relative to their own maxima): the heads 2 t4 and 2 t4 + 1 of a fragment.
struct Merged {
  float4 o;             // head 2 t4: dim d, head 2 t4 + 1: dim d, then both at dim d + 1
  float M0, L0, M1, L1;
};
__device__ __forceinline__ void merge_begin(Merged& a) {
  a.o = make_float4(0.f, 0.f, 0.f, 0.f);
  a.M0 = a.M1 = kNegFloor;
  a.L0 = a.L1 = 0.f;
}
__device__ __forceinline__ void merge_add(Merged& a, float4 o, float4 ml) {
  const float m0 = fmaxf(a.M0, ml.x), m1 = fmaxf(a.M1, ml.z);
  const float a0 = fast_exp2(a.M0 - m0), b0 = fast_exp2(ml.x - m0);
  const float a1 = fast_exp2(a.M1 - m1), b1 = fast_exp2(ml.z - m1);
  a.o.x = a.o.x * a0 + o.x * b0;
  a.o.y = a.o.y * a1 + o.y * b1;
  a.o.z = a.o.z * a0 + o.z * b0;
  a.o.w = a.o.w * a1 + o.w * b1;
  a.L0 = a.L0 * a0 + ml.y * b0;
  a.L1 = a.L1 * a1 + ml.w * b1;
  a.M0 = m0;
  a.M1 = m1;
}
// Normalised result of a fragment to o and lse.  NaN passes on.  Sequences without a token own no tile and do not come here: a
// sum of 0 means that every score was below kNegFloor (-infinity, where 32 bits do not hold it) and gives NaN.
template <int D, typename TO>
__device__ __forceinline__ void emit(const Int4DecodeParams& p, const Merged& a, int b, int head0, int n_heads, int frag,
                                     int lane) {
  constexpr int kSteps = D / 16, kMine = D / 8;
  const int h = (frag / kSteps) * 8 + (lane & 3) * 2, d = kMine * (lane >> 2) + 2 * (frag % kSteps);
  const size_t row = size_t(b) * p.heads + head0 + h;
  TO* o = static_cast<TO*>(p.o) + row * D + d;
  if (h < n_heads) {
    const float inv = a.L0 == 0.f ? NAN : 1.f / a.L0;
    store_out<TO>(o, a.o.x * inv);
    store_out<TO>(o + 1, a.o.z * inv);
    if (d == 0 && p.lse) p.lse[row] = a.L0 == 0.f ? NAN : a.M0 + log2f(a.L0);
  }
  if (h + 1 < n_heads) {
    const float inv = a.L1 == 0.f ? NAN : 1.f / a.L1;
    store_out<TO>(o + D, a.o.y * inv);
    store_out<TO>(o + D + 1, a.o.w * inv);
    if (d == 0 && p.lse) p.lse[row + 1] = a.L1 == 0.f ? NAN : a.M1 + log2f(a.L1);
  }
}

// T: type of q.  NT: head tiles of 8 (a KV head with 9 to 16 q heads has two).  kPair: at most 4 q heads of a KV head, so
// that the second four columns of K's product take the second digit of q, and a lane one token's scores of a record, not two.
template <int D, int NT, bool kPair, typename T, typename TO>
__global__ void __launch_bounds__(kAllThreads, Cfg<D, NT>::kBlocks) gqa_decode_int4_kernel(Int4DecodeParams p) {
  using C = Cfg<D, NT>;
  constexpr int R = C::R;
  constexpr int kKSteps = D / 16;
  constexpr int kKWords = D / 32;      // 32-bit words of a K row that a lane reads: 8 dims each, one k step of 32
  constexpr int kDigits = std::is_same<T, __half>::value ? 3 : 2;   // signed bytes of a q
  constexpr int kDots = kPair ? kDigits - 1 : kDigits;              // products they take
  constexpr int kRows = kPair ? 1 : 2;                              // tokens of a record whose scores a lane has
  static_assert(!kPair || NT == 1, "four heads are one tile");
  constexpr int kVWords = D / 64;      // of a V row
  extern __shared__ __align__(128) unsigned char smem[];
  const uint32_t sbase = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::bars);
  auto bar_full = [&](int s) { return smem_u32(bars + s); };
  auto bar_empty = [&](int s) { return smem_u32(bars + C::kStages + s); };
  auto bar_item_full = [&](int s) { return smem_u32(bars + 2 * C::kStages + s); };
  auto bar_item_empty = [&](int s) { return smem_u32(bars + 2 * C::kStages + kItemSlots + s); };
  const uint32_t bar_dump = smem_u32(bars + 2 * C::kStages + 2 * kItemSlots);         // every warp has left its part of a segment
  const uint32_t bar_merged = smem_u32(bars + 2 * C::kStages + 2 * kItemSlots + 1);   // every warp has merged its share of it
  int* s_misc = reinterpret_cast<int*>(smem + C::misc);    // [0] abort, [6], [7] tickets, [8..11] ragged, [12..19] sums
  volatile int* s_abort = s_misc;
  int* s_prefix = reinterpret_cast<int*>(smem + C::plan);
  int* s_lens = s_prefix + p.batch + 1;
  int* status = p.counters + 2;

  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), kWarps);
    }
    for (int s = 0; s < kItemSlots; ++s) {
      mbar_init(bar_item_full(s), 1);
      mbar_init(bar_item_empty(s), kMathThreads);   // every math thread arrives: an arrival orders its own reads only
    }
    mbar_init(bar_dump, kMathThreads);
    mbar_init(bar_merged, kMathThreads);
    s_misc[0] = 0;
    mbar_fence_init();
  }
  if (warp < kWarps) tile_plan<C::kTile, C::kSegmentCost>(p, tid, s_prefix, s_lens, s_misc + 12, s_misc + 8);
  __syncthreads();

  // Units per range: an equal share per block, but no run shorter than kMinRun tiles (a run costs its partial result's way
  // through memory, and the merge of a lane reads all of them).  Sequences of equal length are cut at whole lanes, or at
  // equal parts of lanes, without gaps, where that leaves the blocks busy to within a twentieth: fewer runs to merge.
  const unsigned lanes = unsigned(p.heads_kv) * unsigned(p.n_hb), lanes_total = unsigned(p.batch) * lanes;
  const bool ragged = s_misc[8] | s_misc[9] | s_misc[10] | s_misc[11];
  const unsigned L = ragged ? 0 : unsigned(s_prefix[1]);
  unsigned gap = C::kSegmentCost, even = L > 0 ? L + gap : 0;
  unsigned total_units = L > 0 ? even * lanes_total : unsigned(s_prefix[p.batch]) * lanes;
  unsigned per = max((total_units + gridDim.x - 1) / gridDim.x, C::kMinRun);
  if (p.force_chunk > 0) {
    // never so short that the ranges outnumber the slots of the workspace (2 per range), nor that one lies in a gap
    per = max(max(unsigned(p.force_chunk), gap + 1), (2u * total_units + unsigned(p.max_slots) - 1) / unsigned(p.max_slots));
  } else if (L > 0) {
    unsigned share = max((L * lanes_total + gridDim.x - 1) / gridDim.x, C::kMinRun);
    unsigned fit = 0;
    if (lanes_total >= gridDim.x) {
      fit = (lanes_total + gridDim.x - 1) / gridDim.x * L;
    } else if (L <= share) {
      fit = share = L;
    } else {
      for (unsigned k = min((L + share - 1) / share, gridDim.x / lanes_total), i = 0; k > 1 && i < 4 && !fit; --k, ++i) {
        const unsigned part = (L + k - 1) / k;
        if (L % part == 0) fit = part;
      }
    }
    if (fit && 20ull * fit <= 21ull * share) {
      per = fit;
      gap = 0;
      even = L;
      total_units = L * lanes_total;
    }
  }
  const long long limit = p.wait_cycles;

  if (warp == kWarps) {
    // ================= producer: q rows and records of this block's segments =================
    constexpr int kRound = 32 / C::kRecords;     // tiles per round: lane l looks up record l % kRecords of tile l / kRecords
    const int my_tile = lane / C::kRecords, my_rec = lane % C::kRecords;
    int stage = 0, round = 0;
    uint32_t stage_par = 0;
    bool alive = true;
    for (int range = blockIdx.x; alive && (unsigned long long)range * per < total_units; range += gridDim.x) {
      const unsigned range_begin = unsigned(range) * per, range_end = min(range_begin + per, total_units);
      for (unsigned u = range_begin; alive && u < range_end; ++round) {
        const int slot = round & 1;
        const uint32_t slot_par = (round >> 1) & 1;
        int ok = 1;
        if (lane == 0) ok = mbar_wait(bar_item_empty(slot), slot_par ^ 1, s_abort, status, 601, limit, 100) ? 1 : 0;
        if (!__shfl_sync(0xffffffffu, ok, 0)) { alive = false; break; }
        const Segment d = segment_at(p, u, range_begin, range_end, range, per, gap, even, s_prefix, s_lens);
        u = d.next;
        if (lane == 0) {
          *reinterpret_cast<Segment*>(smem + C::segs + slot * 64) = d;     // the math warps need not work it out again
          const int head0 = d.hk * p.group + d.hbi * p.hb;
          const uint32_t q_bytes = uint32_t(min(p.hb, p.group - d.hbi * p.hb)) * D * 2;
          mbar_expect_tx(bar_item_full(slot), q_bytes);
          bulk_load(sbase + C::qslots + slot * C::kQSlotBytes,
                    static_cast<const unsigned char*>(p.q) + (size_t(d.b) * p.heads + head0) * D * 2, q_bytes,
                    bar_item_full(slot));
        }
        const int32_t* row = p.table + d.b * p.table_stride;
        const int per_copy = p.records_per_copy;      // (a power of two that divides a page and a tile)
        for (int t0 = d.tile0; t0 < d.tile1 && alive; t0 += kRound) {
          // this lane's copy of the round: its record and the live ones of the per_copy - 1 behind it
          const int t = t0 + my_tile;
          const int token = (t * C::kRecords + my_rec) * kInt4Tokens;
          const bool mine = my_tile < kRound && t < d.tile1 && token < d.len && (my_rec & (per_copy - 1)) == 0;
          const unsigned char* src = nullptr;
          uint32_t bytes = 0;
          bool known = true;
          if (mine) {
            const int column = token / p.page_size, page = row[column];
            known = page >= 0 && page < p.pool_pages && !d.too_long;
            if (known) {
              src = p.pages + ((size_t(page) * p.heads_kv + d.hk) * size_t(p.page_size / kInt4Tokens) +
                               (token - column * p.page_size) / kInt4Tokens) * size_t(C::kRec);
              const int n = min(per_copy, (d.len - token + kInt4Tokens - 1) / kInt4Tokens);
              bytes = uint32_t(n) * C::kRec;
            }
          }
          const bool all_known = __all_sync(0xffffffffu, known);
          const int n_tiles = min(kRound, d.tile1 - t0);
          for (int i = 0; i < n_tiles; ++i) {
            const uint32_t tile_bytes = __reduce_add_sync(0xffffffffu, my_tile == i ? bytes : 0u);
            if (lane == 0) {
              ok = mbar_wait(bar_empty(stage), stage_par ^ 1, s_abort, status, 601, limit, 100) ? 1 : 0;
            }
            if (!__shfl_sync(0xffffffffu, ok, 0)) { alive = false; break; }
            const int at = C::ring + stage * C::kStageBytes + my_rec * C::kRec;
            if (!all_known) {
              // a page outside the pool: nothing is fetched, and the parameters become NaN, which makes the output NaN
              if (my_tile == i && !known)
                for (int r = 0; r < per_copy; ++r)
                  for (int x = 0; x < kInt4Tokens * 8; x += 4)
                    *reinterpret_cast<uint32_t*>(smem + at + r * C::kRec + kInt4Tokens * D + x) = 0x7e007e00u;
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before a later copy into the same place
              __threadfence_block();
              __syncwarp();
            }
            if (lane == 0) mbar_expect_tx(bar_full(stage), tile_bytes);
            __syncwarp();
            if (my_tile == i && bytes > 0) bulk_load(sbase + at, src, bytes, bar_full(stage));
            if (++stage == C::kStages) { stage = 0; stage_par ^= 1; }
          }
        }
      }
    }
  } else {
    // ================= math warps =================
    const int g8 = lane >> 2, t4 = lane & 3;      // "groupID", "threadID_in_group" of the mma fragment layouts
    // token of MMA row 2u is u, of row 2u + 1 it is 4 + (u ^ 3)
    const int u8 = g8 >> 1;
    const int tau = (g8 & 1) ? 4 + (u8 ^ 3) : u8;
    const int k_off = tau * (D / 2) + t4 * (D / 8);                        // K row of MMA row g8; + 8 rows for g8 + 8
    const int v_off0 = 8 * D + t4 * (D / 2) + g8 * (D / 16);               // V row of token t4 (k = 2 t4)
    const int v_off1 = 8 * D + (4 + (t4 ^ 3)) * (D / 2) + g8 * (D / 16);   // V row of k = 2 t4 + 1
    // (kPair) lanes 0 and 1 of a group take token tau of a record and 2 and 3 token tau + 8, of heads 2 (t4 & 1) and the next
    const bool upper = kPair && t4 >= 2;
    const int t_head = kPair ? 2 * (t4 & 1) : 2 * t4, my_tau = tau + (upper ? 8 : 0);
    const int par_off = 16 * D + my_tau * 8;
    const float score_scale = p.softcap > 0.f ? p.sm_scale : p.sm_scale * kLog2e;
    const float inv_cap = p.softcap > 0.f ? 1.f / p.softcap : 0.f;

    float4* s_dump = reinterpret_cast<float4*>(smem + C::dump);
    float4* s_ml = reinterpret_cast<float4*>(smem + C::ml);
    Segment* s_ends = reinterpret_cast<Segment*>(smem + C::ends);
    bool alive = true;
    // Barriers of the math warps with a bounded wait; every thread arrives, since an arrival releases the arriving
    // thread's own stores only.
    uint32_t dump_par = 0, merged_par = 1;     // the dump area starts out free
    auto wait_dump = [&]() -> bool {
      if (!mbar_wait_warp(bar_dump, dump_par, s_abort, status, 603, limit)) { alive = false; return false; }
      dump_par ^= 1;
      return true;
    };
    auto wait_merged = [&]() -> bool {
      if (!mbar_wait_warp(bar_merged, merged_par, s_abort, status, 603, limit)) { alive = false; return false; }
      merged_par ^= 1;
      return true;
    };

    int stage = 0, round = 0;
    uint32_t stage_par = 0;
    for (int range = blockIdx.x; alive && (unsigned long long)range * per < total_units; range += gridDim.x) {
      const unsigned range_begin = unsigned(range) * per, range_end = min(range_begin + per, total_units);
      bool shared = false;
      for (unsigned u = range_begin; alive && u < range_end; ++round) {
        const int slot = round & 1;
        const bool first = u == range_begin;
        if (!mbar_wait_warp(bar_item_full(slot), (round >> 1) & 1, s_abort, status, 602, limit)) { alive = false; break; }
        const Segment& d = *reinterpret_cast<const Segment*>(smem + C::segs + slot * 64);
        u = d.next;
        const int n_heads = min(p.hb, p.group - d.hbi * p.hb), tile0 = d.tile0, tile1 = d.tile1, len = d.len;
        if (tid == 0) s_ends[2] = d;         // (of this thread alone)

        // ---- q: B fragments of S^T = K Q^T as signed bytes; alpha undoes the scale, beta is scale * sum(q) ----
        uint32_t qf[NT][kKWords][kDots][2];
        float alpha[NT][2], beta[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int h = kPair ? g8 & 3 : nt * 8 + g8;
          uint32_t raw[D / 8];       // 16-bit pairs: this lane's D / 4 dims
          const uint4* qs = reinterpret_cast<const uint4*>(smem + C::qslots + slot * C::kQSlotBytes + (h * D + t4 * (D / 4)) * 2);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const uint4 u4 = h < n_heads ? qs[i] : make_uint4(0u, 0u, 0u, 0u);
            raw[4 * i] = u4.x; raw[4 * i + 1] = u4.y; raw[4 * i + 2] = u4.z; raw[4 * i + 3] = u4.w;
          }
          float top = abs_max<T, D / 8>(raw);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // largest |n| in [2^13, 2^14), or [2^20, 2^21): below what the digits and the 22 bits of the sum hold.  The largest
          // finite bf16 asks for e = -114; a head whose largest |q| is below 2^-97 gets fewer bits than that.
          const int e = min(max((kDigits == 3 ? 20 : 13) + 127 - int(__float_as_uint(top) >> 23), -114), 110);
          const float up = pow2f(e);
          // n = rint(q 2^e) as the low bits of 1.5 * 2^23 + n; with 128 (and 128 * 256) added its bytes are the signed
          // digits, of which the lower ones lie 128 too high
          constexpr float kMagic = 12582912.f + (kDigits == 3 ? 32896.f : 128.f);
          int total[kDigits];
          bool finite = true;
#pragma unroll
          for (int digit = 0; digit < kDigits; ++digit) total[digit] = 0;
#pragma unroll
          for (int w = 0; w < kKWords; ++w) {
            uint32_t n[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 x = unpack2<T>(raw[4 * w + i]);
              const float a = fmaf(x.x, up, kMagic), b = fmaf(x.y, up, kMagic);
              finite = finite && a - a == 0.f && b - b == 0.f;
              n[2 * i] = __float_as_uint(a);
              n[2 * i + 1] = __float_as_uint(b);
            }
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {     // dims 0, 2, 4, 6 of a word are its low nibbles, 1, 3, 5, 7 the high ones
              const uint32_t lo = prmt(n[odd], n[2 + odd], 0x5140u), hi = prmt(n[4 + odd], n[6 + odd], 0x5140u);
              uint32_t digit[kDigits];
              digit[0] = prmt(lo, hi, 0x5410u) ^ 0x80808080u;
              digit[1] = prmt(lo, hi, 0x7632u);
              if constexpr (kDigits == 3) {
                digit[1] ^= 0x80808080u;
                // the third byte is 64 + digit, in 7 bits
                const uint32_t d = prmt(prmt(n[odd], n[2 + odd], 0x0062u), prmt(n[4 + odd], n[6 + odd], 0x0062u), 0x5410u) ^ 0x40404040u;
                digit[kDigits - 1] = (d & 0x7f7f7f7fu) | ((d & 0x40404040u) << 1);
              }
#pragma unroll
              for (int i = 0; i < kDigits; ++i) total[i] = __dp4a(int(digit[i]), 0x01010101, total[i]);
              if constexpr (kPair) {
                qf[nt][w][0][odd] = g8 < 4 ? digit[0] : digit[1];
                if constexpr (kDigits == 3) qf[nt][w][kDots - 1][odd] = digit[kDigits - 1];     // in both halves
              } else {
#pragma unroll
                for (int i = 0; i < kDigits; ++i) qf[nt][w][i][odd] = digit[i];
              }
            }
          }
          float sum = float(total[1] * 256 + total[0]);
          if constexpr (kDigits == 3) sum = fmaf(float(total[kDigits - 1]), 65536.f, sum);
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          // an infinity or a NaN of q has no integer: it makes the head's scores NaN
          const unsigned odd_ones = __ballot_sync(0xffffffffu, !finite) >> (lane & 28);
          const float a = (odd_ones & 15u) ? NAN : score_scale * pow2f(-e), bsum = a * sum;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            alpha[nt][i] = __shfl_sync(0xffffffffu, a, (t_head + i) * 4);
            beta[nt][i] = __shfl_sync(0xffffffffu, bsum, (t_head + i) * 4);
          }
        }
        mbar_arrive(bar_item_empty(slot));   // q is in registers (every thread: its own reads)

        float oacc[NT][kKSteps][4], wacc[NT][4];         // wacc: 7.5 * sum of the rounded weights, in every row
        float m_run[NT][2], l_run[NT][2], corr[NT][2];   // corr: sum of p * vm
        int v_exp = -24;                                 // |vs| <= 2^v_exp so far (the smallest subnormal's exponent)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) { m_run[nt][i] = kNegFloor; l_run[nt][i] = 0.f; corr[nt][i] = 0.f; }
#pragma unroll
          for (int mt = 0; mt < kKSteps; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) oacc[nt][mt][e] = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) wacc[nt][e] = 0.f;
        }

        for (int tile = tile0; tile < tile1; ++tile) {
          if (!mbar_wait_warp(bar_full(stage), stage_par, s_abort, status, 602, limit)) { alive = false; break; }
          const unsigned char* st = smem + C::ring + stage * C::kStageBytes + warp * C::kRec;
          const int tok0 = (tile * C::kRecords + warp) * kInt4Tokens + my_tau;

          // ---- S^T = K Q^T on the codes: 16 tokens x 8 heads per record; the records' products interleave, since each
          //      accumulator is a chain of kKWords dependent MMAs ----
          float x[R][NT][2 * kRows];           // scores (log2): two heads of each token
          float vs[R][kRows], vm[R][kRows];    // V scale, and value of the middle code 7.5
          {
            uint32_t ka[R][kKWords], kb[R][kKWords];
#pragma unroll
            for (int j = 0; j < R; ++j) {
              lds_words<kKWords>(ka[j], (st + j * kWarps * C::kRec) + k_off);
              lds_words<kKWords>(kb[j], (st + j * kWarps * C::kRec) + k_off + 4 * D);
            }
            int dot[R][NT][kDots][4];
#pragma unroll
            for (int w = 0; w < kKWords; ++w) {
#pragma unroll
              for (int j = 0; j < R; ++j) {
                const uint32_t a[4] = {ka[j][w] & 0x0f0f0f0fu, kb[j][w] & 0x0f0f0f0fu, (ka[j][w] >> 4) & 0x0f0f0f0fu,
                                       (kb[j][w] >> 4) & 0x0f0f0f0fu};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int digit = 0; digit < kDots; ++digit)
                    mma_16832_u8s8(dot[j][nt][digit], a, qf[nt][w][digit], w == 0);
              }
            }
#pragma unroll
            for (int j = 0; j < R; ++j) {
              float ks[kRows], km[kRows];
#pragma unroll
              for (int i = 0; i < kRows; ++i) {
                const uint2 params = *reinterpret_cast<const uint2*>((st + j * kWarps * C::kRec) + par_off + 64 * i);
                const float2 kp = f16x2_to_f32x2(params.x), vp = f16x2_to_f32x2(params.y);
                ks[i] = kp.x; km[i] = kp.y;
                vs[j][i] = vp.x; vm[j][i] = fmaf(7.5f, vp.x, vp.y);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2 * kRows; ++e) {
                  int n, third = 0;
                  if constexpr (kPair) {
                    // this lane's digit of its own token, and the other one, which is what the lane two further on does
                    // not need
                    const int own = upper ? dot[j][nt][0][2 + e] : dot[j][nt][0][e];
                    const int other = __shfl_xor_sync(0xffffffffu, upper ? dot[j][nt][0][e] : dot[j][nt][0][2 + e], 2);
                    n = own * (upper ? 256 : 1) + other * (upper ? 1 : 256);
                    if constexpr (kDigits == 3) third = upper ? dot[j][nt][kDots - 1][2 + e] : dot[j][nt][kDots - 1][e];
                  } else {
                    n = dot[j][nt][kDots > 1 ? 1 : 0][e] * 256 + dot[j][nt][0][e];
                    if constexpr (kDigits == 3) third = dot[j][nt][kDots - 1][e];
                  }
                  float s = float(n);
                  if constexpr (kDigits == 3) s = fmaf(float(third), 65536.f, s);
                  x[j][nt][e] = fmaf(s * alpha[nt][e & 1], ks[e >> 1], km[e >> 1] * beta[nt][e & 1]);
                }
              }
            }
            if (p.softcap > 0.f) {
#pragma unroll
              for (int j = 0; j < R; ++j)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int e = 0; e < 2 * kRows; ++e) x[j][nt][e] = soft_cap(x[j][nt][e], p.softcap, inv_cap) * kLog2e;
            }
          }
          if ((tile + 1) * C::kTile > len) {
            // tokens behind the end: whatever their place holds (NaN, or an older tile) stays out of every sum
#pragma unroll
            for (int j = 0; j < R; ++j) {
#pragma unroll
              for (int i = 0; i < kRows; ++i) {
                if (tok0 + j * kWarps * kInt4Tokens + 8 * i >= len) {
                  vs[j][i] = 0.f;
                  vm[j][i] = 0.f;
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) { x[j][nt][2 * i] = -INFINITY; x[j][nt][2 * i + 1] = -INFINITY; }
                }
              }
            }
          }

          // ---- running maximum and V scale: moved only when a token exceeds them ----
          float mx[NT][2], vtop = 0.f;
          bool grow = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              mx[nt][i] = -INFINITY;
#pragma unroll
              for (int j = 0; j < R; ++j)
                mx[nt][i] = kPair ? fmaxf(mx[nt][i], x[j][nt][i]) : max3(mx[nt][i], x[j][nt][i], x[j][nt][2 * (kRows - 1) + i]);
              grow |= mx[nt][i] > m_run[nt][i] + kGrow;
            }
          }
#pragma unroll
          for (int j = 0; j < R; ++j) vtop = max3(vtop, fabsf(vs[j][0]), fabsf(vs[j][kRows - 1]));
          grow |= vtop > pow2f(v_exp);
          if (__any_sync(0xffffffffu, grow)) {
            const uint32_t bits = __float_as_uint(vtop);
            const uint32_t top = __reduce_max_sync(0xffffffffu, bits < 0x7f800000u ? bits : 0u);
            const int e_new = max(v_exp, int(top >> 23) - 126);     // 2^e_new is above every |vs| so far
            const float down = e_new == v_exp ? 1.f : pow2f(max(v_exp - e_new, -126));
            v_exp = e_new;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float al[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float m = mx[nt][i];
#pragma unroll
                for (int o = kPair ? 2 : 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                m = fmaxf(m_run[nt][i], m);
                al[i] = fast_exp2(m_run[nt][i] - m);
                m_run[nt][i] = m;
                l_run[nt][i] *= al[i];
                corr[nt][i] *= al[i];
                al[i] *= down;
              }
#pragma unroll
              for (int mt = 0; mt < kKSteps; ++mt) {
                oacc[nt][mt][0] *= al[0]; oacc[nt][mt][1] *= al[1];
                oacc[nt][mt][2] *= al[0]; oacc[nt][mt][3] *= al[1];
              }
              wacc[nt][0] *= al[0]; wacc[nt][1] *= al[1];
            }
          }

          // ---- P, and O^T += V^T (P vs)^T on the codes ----
          const float v_norm = pow2f(kPBits - v_exp);
#pragma unroll
          for (int j = 0; j < R; ++j) {
            uint32_t pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
              for (int i = 0; i < kRows; ++i) {
                const float p0 = fast_exp2(x[j][nt][2 * i] - m_run[nt][0]), p1 = fast_exp2(x[j][nt][2 * i + 1] - m_run[nt][1]);
                l_run[nt][0] += p0;
                l_run[nt][1] += p1;
                corr[nt][0] = fmaf(p0, vm[j][i], corr[nt][0]);
                corr[nt][1] = fmaf(p1, vm[j][i], corr[nt][1]);
                const float scale = vs[j][i] * v_norm;
                pb[nt][i] = movmatrix_trans(pack2<__half>(p0 * scale, p1 * scale));
              }
              // columns 0..3 now hold tokens 0..7 of the four heads and columns 4..7 tokens 8..15, which the former want too
              // (what the latter add up is not used)
              if constexpr (kPair) pb[nt][1] = __shfl_xor_sync(0xffffffffu, pb[nt][0], 16);
              const uint32_t mid[4] = {kMid, kMid, kMid, kMid};
              mma_16816<__half>(wacc[nt], mid, pb[nt]);
            }
            const unsigned char* rec = st + j * kWarps * C::kRec;
            uint32_t v0[kVWords], v1[kVWords], v2[kVWords], v3[kVWords];
            lds_words<kVWords>(v0, rec + v_off0);
            lds_words<kVWords>(v1, rec + v_off1);
            lds_words<kVWords>(v2, rec + v_off0 + 4 * D);
            lds_words<kVWords>(v3, rec + v_off1 + 4 * D);
#pragma unroll
            for (int w = 0; w < kVWords; ++w) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                // four dims of two tokens each: m-tiles 4 w + 2 half and the next
                const uint32_t a = prmt(v0[w], v1[w], half ? 0x7632u : 0x5410u);
                const uint32_t b = prmt(v2[w], v3[w], half ? 0x7632u : 0x5410u);
                // (rows g8: n0, rows g8 + 8: n0 + 16 n1)
                const uint32_t ha = prmt(a, 0u, 0x4341u), hb = prmt(b, 0u, 0x4341u);
                const uint32_t a0[4] = {a & 0x000f000fu, a & 0x00ff00ffu, b & 0x000f000fu, b & 0x00ff00ffu};
                const uint32_t a1[4] = {ha & 0x000f000fu, ha, hb & 0x000f000fu, hb};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  mma_16816<__half>(oacc[nt][4 * w + 2 * half], a0, pb[nt]);
                  mma_16816<__half>(oacc[nt][4 * w + 2 * half + 1], a1, pb[nt]);
                }
              }
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_empty(stage));
          if (++stage == C::kStages) { stage = 0; stage_par ^= 1; }
        }
        if (!alive) break;

        // ---- the warps meet: (max, sum, O) relative to each warp's maximum through shared memory ----
        const float unit_lo = pow2f(24 - kPBits) * pow2f(v_exp), unit_hi = pow2f(20 - kPBits) * pow2f(v_exp);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int o = kPair ? 2 : 4; o < 32; o <<= 1) {
              l_run[nt][i] += __shfl_xor_sync(0xffffffffu, l_run[nt][i], o);
              corr[nt][i] += __shfl_xor_sync(0xffffffffu, corr[nt][i], o);
            }
            corr[nt][i] = fmaf(-wacc[nt][i], unit_lo * 5.9604644775390625e-8f, corr[nt][i]);   // 2^-24: wacc is in whole codes
          }
        }
        if (!wait_merged()) break;      // the area held the previous segment
        if (tid == 0) {
          if (first) s_ends[0] = s_ends[2];
          s_ends[1] = s_ends[2];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int mt = 0; mt < kKSteps; ++mt) {
            float4 v;
            v.x = fmaf(oacc[nt][mt][0], unit_lo, corr[nt][0]);
            v.y = fmaf(oacc[nt][mt][1], unit_lo, corr[nt][1]);
            v.z = fmaf(oacc[nt][mt][2] - oacc[nt][mt][0], unit_hi, corr[nt][0]);
            v.w = fmaf(oacc[nt][mt][3] - oacc[nt][mt][1], unit_hi, corr[nt][1]);
            s_dump[(warp * C::kFrags + nt * kKSteps + mt) * 32 + lane] = v;
          }
          if (g8 == 0) s_ml[(warp * NT + nt) * 4 + t4] = make_float4(m_run[nt][0], l_run[nt][0], m_run[nt][1], l_run[nt][1]);
        }
        mbar_arrive(bar_dump);
        if (!wait_dump()) break;
        const Segment e = s_ends[1];
#pragma unroll
        for (int f = warp; f < C::kFrags; f += kWarps) {
          const int nt = f / kKSteps;
          Merged a;
          merge_begin(a);
#pragma unroll
          for (int w = 0; w < kWarps; ++w)
            merge_add(a, s_dump[(w * C::kFrags + f) * 32 + lane], s_ml[(w * NT + nt) * 4 + t4]);
          if (e.n_runs == 1) {
            emit<D, TO>(p, a, e.b, e.hk * p.group + e.hbi * p.hb, min(p.hb, p.group - e.hbi * p.hb), f, lane);
          } else {
            p.part_o[(size_t(e.slot) * C::kFrags + f) * 32 + lane] = a.o;
            if (f % kKSteps == 0 && g8 == 0)
              p.part_ml[(size_t(e.slot) * NT + nt) * 4 + t4] = make_float4(a.M0, a.L0, a.M1, a.L1);
          }
        }
        shared = s_ends[0].n_runs > 1 || e.n_runs > 1;      // (the range's first segment, its last so far)
        mbar_arrive(bar_merged);
      }
      if (!alive) break;
      // ---- end of the range: only its first and last segments can share their lanes with other ranges; the last block to
      //      finish such a lane merges it ----
      if (!shared) continue;
      if (!wait_merged()) break;          // every warp's partial results are written
      if (lane == 0 && warp < 2) {        // one thread takes the first segment's ticket, another the last one's
        const Segment& d = s_ends[warp];
        int mine = 0;
        if (d.n_runs > 1 && (warp == 0 || d.lane != s_ends[0].lane)) {
          int* at = p.counters + kCounterWords + d.lane;
          int n;
          asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(n) : "l"(at) : "memory");
          if (n == d.n_runs - 1) {
            *at = 0;      // zero again for the next launch
            mine = 1;
          }
        }
        s_misc[6 + warp] = mine;
      }
      mbar_arrive(bar_dump);
      if (!wait_dump()) break;
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        if (!s_misc[6 + i]) continue;
        const Segment d = s_ends[i];
        // A warp merges fragments of one head tile side by side and has the loads of kBatch runs in flight: a long lane cut
        // over all SMs has dozens, and their latency would add up.
        constexpr int kSide = kKSteps / kWarps, kBatch = 6;
        for (int f0 = warp; f0 < C::kFrags; f0 += kSide * kWarps) {
          Merged a[kSide];
#pragma unroll
          for (int s = 0; s < kSide; ++s) merge_begin(a[s]);
          for (int r0 = 0; r0 < d.n_runs; r0 += kBatch) {
            float4 o[kBatch][kSide], ml[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
              const int r = min(r0 + i, d.n_runs - 1);
              const size_t it = size_t(segment_slot(d.first_range + r, per, d.lane_start));
              ml[i] = __ldcg(p.part_ml + (it * NT + f0 / kKSteps) * 4 + t4);
#pragma unroll
              for (int s = 0; s < kSide; ++s) o[i][s] = __ldcg(p.part_o + (it * C::kFrags + f0 + s * kWarps) * 32 + lane);
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
              if (r0 + i < d.n_runs) {
#pragma unroll
                for (int s = 0; s < kSide; ++s) merge_add(a[s], o[i][s], ml[i]);
              }
          }
          const int head0 = d.hk * p.group + d.hbi * p.hb, n_heads = min(p.hb, p.group - d.hbi * p.hb);
#pragma unroll
          for (int s = 0; s < kSide; ++s) emit<D, TO>(p, a[s], d.b, head0, n_heads, f0 + s * kWarps, lane);
        }
      }
      mbar_arrive(bar_merged);            // the tickets' words and the dump area are free again
    }
    // sequences without a token own no tile
    if (alive) {
      for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        if (s_prefix[b + 1] != s_prefix[b]) continue;
        for (int idx = tid; idx < p.heads * D; idx += kMathThreads) {
          store_out<TO>(static_cast<TO*>(p.o) + size_t(b) * p.heads * D + idx, 0.f);
          if (idx < p.heads && p.lse) p.lse[size_t(b) * p.heads + idx] = -INFINITY;
        }
      }
    }
  }
  if (*s_abort) {
    // copies still in flight land before the shared memory is released
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
}

// ---- host side -------------------------------------------------------------------------------------------------------
struct Int4Layout {
  int hb, n_hb, nt, max_slots;
  size_t counters_bytes, part_o_bytes, total;
};
Int4Layout make_layout(int batch, int heads, int heads_kv, int dim) {
  Int4Layout L{};
  const int group = heads / heads_kv;
  L.hb = group < 16 ? group : 16;
  L.nt = L.hb <= 8 ? 1 : 2;
  L.n_hb = (group + L.hb - 1) / L.hb;
  L.max_slots = sm_count() * kSlotsPerSm;
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  L.counters_bytes = up((kCounterWords + size_t(batch) * heads_kv * L.n_hb) * 4);
  L.part_o_bytes = up(size_t(L.max_slots) * L.nt * 8 * dim * 4);
  L.total = L.counters_bytes + L.part_o_bytes + up(size_t(L.max_slots) * L.nt * 8 * 2 * 4);
  return L;
}

template <int D, int NT, bool kPair, typename T, typename TO>
int launch(const Int4DecodeParams& p, cudaStream_t stream) {
  auto kern = gqa_decode_int4_kernel<D, NT, kPair, T, TO>;
  const size_t smem = smem_bytes<D, NT>(p.batch);
  static thread_local bool configured[64] = {false};
  static thread_local size_t sized_for[64] = {0};
  static thread_local int resident[64] = {0};
  int dev = 0;
  TB200_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) TB200_FAIL(TB200_ERR_UNSUPPORTED, "device index %d", dev);
  if (!configured[dev]) {
    // The limit belongs to the function, not to this thread: every thread sets the one that the largest batch needs, so
    // that none takes it from another.
    TB200_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem_bytes<D, NT>(kMaxBatch))));
    configured[dev] = true;
  }
  if (sized_for[dev] != smem) {
    int n = 0;
    TB200_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kAllThreads, smem));
    if (n < 1) TB200_FAIL(TB200_ERR_UNSUPPORTED, "a batch of %d needs more shared memory than a block has", p.batch);
    resident[dev] = n < Cfg<D, NT>::kBlocks ? n : Cfg<D, NT>::kBlocks;
    sized_for[dev] = smem;
  }
  kern<<<sm_count() * resident[dev], kAllThreads, smem, stream>>>(p);
  TB200_CUDA_CHECK(cudaGetLastError());
  return TB200_OK;
}
template <int D, typename T, typename TO>
int launch_nt(const Int4DecodeParams& p, int nt, cudaStream_t s) {
  if (nt == 2) return launch<D, 2, false, T, TO>(p, s);
  return p.hb <= 4 ? launch<D, 1, true, T, TO>(p, s) : launch<D, 1, false, T, TO>(p, s);
}
template <int D, typename T>
int launch_o(const Int4DecodeParams& p, int nt, int o_dtype, cudaStream_t s) {
  if (o_dtype == TB200_F32) return launch_nt<D, T, float>(p, nt, s);
  if (o_dtype == TB200_BF16) return launch_nt<D, T, __nv_bfloat16>(p, nt, s);
  return launch_nt<D, T, __half>(p, nt, s);
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" size_t tb200_gqa_decode_int4_workspace_bytes(int batch, int heads, int heads_kv, int dim) {
  if (batch <= 0 || heads <= 0 || heads_kv <= 0 || heads % heads_kv != 0 || (dim != 64 && dim != 128)) return 0;
  return make_layout(batch, heads, heads_kv, dim).total;
}

extern "C" int tb200_gqa_decode_int4_status(int32_t* code, int reset, void* stream) {
  if (!code) TB200_FAIL(TB200_ERR_BAD_ARGUMENT, "code must be non-null");
  void* word = nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  TB200_CUDA_CHECK(cudaGetSymbolAddress(&word, g_gave_up));
  TB200_CUDA_CHECK(cudaMemcpyAsync(code, word, sizeof(int32_t), cudaMemcpyDeviceToHost, s));
  TB200_CUDA_CHECK(cudaStreamSynchronize(s));
  if (reset && *code) TB200_CUDA_CHECK(cudaMemsetAsync(word, 0, sizeof(int32_t), s));
  return TB200_OK;
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
  if (batch > kMaxBatch) TB200_FAIL(TB200_ERR_UNSUPPORTED, "batch %d exceeds %d", batch, kMaxBatch);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv_pages)) & 15)
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "q and kv_pages must start on 16-byte boundaries");
  const Int4Layout L = make_layout(batch, heads, heads_kv, dim);
  if (workspace_bytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & 255))
    TB200_FAIL(TB200_ERR_WORKSPACE, "workspace must be 256-byte aligned and hold %zu bytes", L.total);
  Int4DecodeParams p{};
  p.q = q; p.pages = static_cast<const unsigned char*>(kv_pages); p.o = o; p.lse = lse; p.lens = real_seqlen_kv;
  p.table = block_table; p.table_stride = block_table_stride; p.table_width = block_table_width;
  p.pool_pages = int(pool_pages); p.batch = batch; p.heads = heads; p.heads_kv = heads_kv; p.group = heads / heads_kv;
  p.page_size = page_size; p.hb = L.hb; p.n_hb = L.n_hb;
  const long long capacity = (long long)block_table_width * page_size;
  p.capacity = int(capacity < 0x7fff0000LL ? capacity : 0x7fff0000LL);
  // the partition counts tiles in 32 bits (tiles of 64 tokens or more, less than 4 for a gap)
  if ((long long)batch * ((p.capacity + 63) / 64 + 4) * heads_kv * L.n_hb >= (1LL << 31))
    TB200_FAIL(TB200_ERR_UNSUPPORTED, "batch x table width x heads_kv is too large");
  p.sm_scale = sm_scale; p.softcap = softcap;
  p.force_chunk = (flags >> TB200_DECODE_CHUNK_TILES_SHIFT) & 0xFFFF;
  p.max_slots = L.max_slots;
  p.counters = static_cast<int*>(workspace);
  p.part_o = reinterpret_cast<float4*>(static_cast<unsigned char*>(workspace) + L.counters_bytes);
  p.part_ml = reinterpret_cast<float4*>(static_cast<unsigned char*>(workspace) + L.counters_bytes + L.part_o_bytes);
  const int wait_log2 = (flags >> TB200_DECODE_WAIT_LOG2_SHIFT) & 31;
  p.wait_cycles = wait_log2 ? 1LL << wait_log2 : 1000000000LL;   // about 0.5 s
  static_assert(Cfg<128, 1>::kRecords == 8 && Cfg<128, 2>::kRecords == 8 && Cfg<64, 1>::kRecords == 8 && Cfg<64, 2>::kRecords == 8,
                "the copies' sizes");
  p.records_per_copy = 1;
  while (p.records_per_copy < 8 && page_size / kInt4Tokens % (2 * p.records_per_copy) == 0) p.records_per_copy *= 2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (q_dtype == TB200_BF16)
    return dim == 64 ? launch_o<64, __nv_bfloat16>(p, L.nt, o_dtype, s) : launch_o<128, __nv_bfloat16>(p, L.nt, o_dtype, s);
  return dim == 64 ? launch_o<64, __half>(p, L.nt, o_dtype, s) : launch_o<128, __half>(p, L.nt, o_dtype, s);
}
