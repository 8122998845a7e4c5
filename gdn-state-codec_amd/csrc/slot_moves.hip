// Copies between the slots of a state cache: the order in which any pairs (source,
// target) can be copied in place, the moves that pack live slots to the front, and the
// copies.
//
// A pair has to be carried out before the pair that overwrites its source, if there is
// one (its successor); every pair has at most one.  The pairs then form trees that end in
// a pair whose source nobody overwrites, and cycles.  A cycle is cut before the pair of
// its lowest number, which first keeps what its target held, and its last pair writes that.
// Ordered by tree and by falling distance from the tree's end, every pair comes before
// its successor, and pairs of different trees share no slot that is written.  Trees whose
// ends read one slot stand side by side, so that a fork's reads after the first come from
// the caches: 300 slots of 32 encoded heads (330 MB, each source once) take 55 us, unsorted 75.
//
// One workgroup finds the order (hash tables and pointer doubling in LDS, a sort): 3.8 us for
// 4 pairs, 9 for a beam step's 96 and 8.5 for 300, barriers and LDS latency; the moves of a
// compaction of 256 slots 4.8.
//
// copy_slots needs no order between threads: a thread owns a run of 16 bytes of every
// slot and carries the rows out in turn, some loads at a time.  A load may come before any
// store (each reads what its slot held before the call), a store never before the loads
// of the rows before it.  Trees are dealt over the grid's second dimension, so that many
// small slots fill the card too.  HBM bounds it: 96 slots of 8 layers' 32 heads (2.7 GB, each
// source once) take 523 us, 5.2 TB/s; 90 moves of a compaction (512 MB) 85 us, 6.0 TB/s.  One
// cycle over many small slots is bound by its own order: 500 slots of 32 KiB take 42 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gdn_state_codec_slots.h"
#include "lane_exchange.h"
#include "launch.h"
#include "stream_memory.h"

namespace gdn {
namespace {

constexpr int kMaxPairs = GDN_STATE_CODEC_MAX_MOVES;
constexpr int kMaxCompacted = GDN_STATE_CODEC_MAX_COMPACTED;
constexpr int kSaves = GDN_STATE_CODEC_MOVE_SAVES;
constexpr int kSaved = GDN_STATE_CODEC_MOVE_SAVED;

// ---------------------------------------------------------------- the order

constexpr int kPlanThreads = 1024;
constexpr int kEach = kMaxPairs / kPlanThreads;
constexpr int kHashed = 2 * kMaxPairs;
constexpr uint64_t kLeftOut = 1ull << 62;  // a key of a pair that is left out, at least

struct Plan {
  int32_t source[kMaxPairs];
  int32_t target[kMaxPairs];
  union {
    int32_t hashed[kHashed];   // pairs by target, then by source; -1 free
    uint64_t key[kMaxPairs];   // to sort pairs by
  };
  int32_t next[kMaxPairs];     // a pair 2^i steps on
  int32_t steps[kMaxPairs];    // how many of them are real
  int32_t lowest[kMaxPairs];   // of the pairs passed
  uint8_t flags[kMaxPairs];
  uint8_t on_cycle[kMaxPairs];
  int chained, cycles, shared;
};

__device__ __forceinline__ uint32_t hash_of(int32_t slot) {
  return (static_cast<uint32_t>(slot) * 2654435761u) >> 16;
}

// The place of `slot` in the table, whose pairs name their slot in `slots`, or of the free
// place where it would be.  At least half of the table's places stay free.
__device__ __forceinline__ uint32_t place_of(const int32_t* hashed, const int32_t* slots,
                                             int32_t slot, uint32_t mask) {
  uint32_t at = hash_of(slot) & mask;
  while (hashed[at] >= 0 && slots[hashed[at]] != slot) at = (at + 1) & mask;
  return at;
}

// Enters pair `pair` of `slot`; of the pairs of one slot the highest stays.
__device__ __forceinline__ void enter(int32_t* hashed, const int32_t* slots, int32_t slot,
                                      int32_t pair, uint32_t mask) {
  uint32_t at = hash_of(slot) & mask;
  while (true) {
    const int before = atomicCAS(&hashed[at], -1, pair);
    if (before < 0) return;
    if (slots[before] == slot) {
      atomicMax(&hashed[at], pair);
      return;
    }
    at = (at + 1) & mask;
  }
}

// next, steps and lowest after 2^rounds >= pairs steps, from one step.
__device__ __forceinline__ void follow(Plan& p, int pairs) {
  for (int reach = 1; reach < pairs; reach <<= 1) {
    int32_t next[kEach], steps[kEach], lowest[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = threadIdx.x + e * blockDim.x;
      if (i >= pairs) break;
      const int n = p.next[i];
      next[e] = p.next[n];
      steps[e] = p.steps[i] + p.steps[n];
      lowest[e] = min(p.lowest[i], p.lowest[n]);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = threadIdx.x + e * blockDim.x;
      if (i >= pairs) break;
      p.next[i] = next[e];
      p.steps[i] = steps[e];
      p.lowest[i] = lowest[e];
    }
    __syncthreads();
  }
}

// x of lane ^ kMask.
template <int kMask>
__device__ __forceinline__ uint64_t partner(uint64_t x, int lane) {
  if constexpr (kMask == 16 || kMask == 32) {
    const bool up = (lane & kMask) != 0;
    const auto low = kMask == 32 ? __builtin_amdgcn_permlane32_swap(x, x, false, false)
                                 : __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const auto high = kMask == 32
        ? __builtin_amdgcn_permlane32_swap(x >> 32, x >> 32, false, false)
        : __builtin_amdgcn_permlane16_swap(x >> 32, x >> 32, false, false);
    const uint32_t low_up = low[0], low_down = low[1], high_up = high[0], high_down = high[1];
    return static_cast<uint64_t>(up ? high_up : high_down) << 32 | (up ? low_up : low_down);
  } else {
    return dpp_xor<kMask>(x);
  }
}

// One step of sorting key[e] of place threadIdx.x + e x blockDim.x, with the keys of the
// places `gap` on.
__device__ __forceinline__ uint64_t sorted(uint64_t key, uint64_t other, int place, int gap,
                                           int run) {
  const bool least = ((place & gap) == 0) == ((place & run) == 0);
  return (key < other) == least ? key : other;
}
template <int kGap>
__device__ __forceinline__ void sort_lanes(uint64_t (&key)[kEach], int run, int size) {
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (e * static_cast<int>(blockDim.x) >= size) break;
    key[e] = sorted(key[e], partner<kGap>(key[e], threadIdx.x), threadIdx.x + e * blockDim.x,
                    kGap, run);
  }
}
// Sorts the first `size` places (a power of two).  Bitonic: keys of one wavefront's places
// are exchanged between lanes, others through `shared` (all through it: 96 pairs' order
// takes 12.5 us, 300 pairs' 13.8).
__device__ __forceinline__ void sort(uint64_t (&key)[kEach], uint64_t* shared, int size) {
  const int t = threadIdx.x, threads = blockDim.x;
  for (int run = 2; run <= size; run <<= 1) {
    for (int gap = run >> 1; gap >= 64; gap >>= 1) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (e * threads < size) shared[t + e * threads] = key[e];
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int place = t + e * threads;
        if (e * threads < size) key[e] = sorted(key[e], shared[place ^ gap], place, gap, run);
      }
      __syncthreads();
    }
    if (run >= 64) sort_lanes<32>(key, run, size);
    if (run >= 32) sort_lanes<16>(key, run, size);
    if (run >= 16) sort_lanes<8>(key, run, size);
    if (run >= 8) sort_lanes<4>(key, run, size);
    if (run >= 4) sort_lanes<2>(key, run, size);
    sort_lanes<1>(key, run, size);
  }
}

// `table`: places of the hash table, a power of two of at least 2 x pairs.
__global__ __launch_bounds__(kPlanThreads) void slot_moves_kernel(
    const int32_t* __restrict__ sources, const int32_t* __restrict__ targets, int pairs,
    uint32_t slots, uint32_t table, int4* __restrict__ steps) {
  __shared__ Plan p;
  const int t = threadIdx.x, threads = blockDim.x;
  const uint32_t mask = table - 1;
  for (uint32_t i = t; i < table; i += threads) p.hashed[i] = -1;
  if (t == 0) p.chained = p.cycles = p.shared = 0;
  for (int i = t; i < pairs; i += threads) {
    const int32_t source = sources[i], target = targets[i];
    const bool counts = static_cast<uint32_t>(target) < slots &&
                        (source == -1 || static_cast<uint32_t>(source) < slots);
    p.source[i] = source;
    p.target[i] = counts ? target : -1;
    p.flags[i] = p.on_cycle[i] = 0;
  }
  __syncthreads();
  for (int i = t; i < pairs; i += threads) {
    if (p.target[i] >= 0) enter(p.hashed, p.target, p.target[i], i, mask);
  }
  __syncthreads();
  bool live[kEach];
  int after[kEach], reads[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = t + e * threads;
    live[e] = false;
    after[e] = reads[e] = -1;
    if (i >= pairs) break;
    // The last pair of a target counts.
    live[e] = p.target[i] >= 0 &&
              p.hashed[place_of(p.hashed, p.target, p.target[i], mask)] == i;
    if (live[e] && p.source[i] >= 0) {
      after[e] = p.hashed[place_of(p.hashed, p.target, p.source[i], mask)];
      if (after[e] == i) after[e] = -1;  // onto itself
    }
    p.next[i] = after[e] >= 0 ? after[e] : i;
    p.steps[i] = after[e] >= 0 ? 1 : 0;
    p.lowest[i] = i;
    if (after[e] >= 0) p.chained = 1;
  }
  __syncthreads();
  // Pairs of one source, which are put side by side: its last pair's number.
  for (uint32_t i = t; i < table; i += threads) p.hashed[i] = -1;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = t + e * threads;
    if (i < pairs && live[e]) enter(p.hashed, p.source, p.source[i], i, mask);
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = t + e * threads;
    if (i >= pairs) break;
    if (live[e]) {
      reads[e] = p.hashed[place_of(p.hashed, p.source, p.source[i], mask)];
      if (reads[e] != i) p.shared = 1;
    }
  }
  __syncthreads();
  if (!p.chained && !p.shared) {  // any order will do
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = t + e * threads;
      if (i >= pairs) break;
      steps[i] = live[e] ? make_int4(p.source[i], p.target[i], 0, i + 1)
                         : make_int4(-1, -1, 0, i + 1);
    }
    return;
  }

  if (p.chained) {
    follow(p, pairs);
    // An end is its own successor; 2^rounds >= pairs real steps are taken only on cycles,
    // and every pair of a cycle is reached by one of its own.
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = t + e * threads;
      if (i >= pairs) break;
      if (p.steps[i] >= pairs) {
        p.on_cycle[p.next[i]] = 1;
        p.cycles = 1;
      }
    }
    __syncthreads();
    if (p.cycles) {
      int head[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int i = t + e * threads;
        head[e] = i < pairs && p.on_cycle[i] ? p.lowest[i] : -1;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int i = t + e * threads;
        if (i >= pairs) break;
        if (head[e] == i) p.flags[i] |= kSaves;
        if (head[e] >= 0 && after[e] == head[e]) {
          p.flags[i] |= kSaved;
          after[e] = -1;
        }
        p.next[i] = after[e] >= 0 ? after[e] : i;
        p.steps[i] = after[e] >= 0 ? 1 : 0;
      }
      __syncthreads();
      follow(p, pairs);
    }
  }

  // Order by what a tree's end reads, by tree (the pair at its end; what is left out last)
  // and by falling distance.  `lowest` takes what each pair reads.
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = t + e * threads;
    if (i < pairs) p.lowest[i] = reads[e];
  }
  __syncthreads();
  int size = 1;
  while (size < pairs) size <<= 1;
  uint64_t key[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = t + e * threads;
    key[e] = ~0ull;
    if (i < pairs) {
      const uint64_t end = p.next[i];
      key[e] = live[e] ? static_cast<uint64_t>(p.lowest[end]) << 48 | end << 32 |
                             static_cast<uint64_t>(kMaxPairs - p.steps[i]) << 16 | i
                       : kLeftOut | i;
    }
  }
  __syncthreads();
  sort(key, p.key, size);
  // A tree's last pair, the one at its end, says where it ends.
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int end = static_cast<int>(key[e] >> 32 & 0xFFFF);
    if (key[e] < kLeftOut && (key[e] & 0xFFFF) == end) p.steps[end] = t + e * threads + 1;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int place = t + e * threads;
    if (place >= pairs) break;
    const int i = static_cast<int>(key[e] & 0xFFFF);
    const int end = static_cast<int>(key[e] >> 32 & 0xFFFF);
    steps[place] = key[e] < kLeftOut
                       ? make_int4(p.source[i], p.target[i], p.flags[i], p.steps[end])
                       : make_int4(-1, -1, 0, place + 1);
  }
}

// --------------------------------------------------------------- compaction

// Sum of the threads before this one; `total` is the workgroup's.
__device__ __forceinline__ int sum_before(int x, int (&waves)[16], int& total) {
  const int lane = threadIdx.x & 63;
  int sum = x;
#pragma unroll
  for (int step = 1; step < 64; step <<= 1) {
    const int other = __shfl_up(sum, step);
    if (lane >= step) sum += other;
  }
  if (lane == 63) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 6)) before += waves[w];
    total += waves[w];
  }
  return before + sum - x;
}

__global__ __launch_bounds__(kPlanThreads) void compaction_kernel(
    const int32_t* __restrict__ live, int slots, int4* __restrict__ steps,
    int32_t* __restrict__ placed, int32_t* __restrict__ count) {
  __shared__ uint16_t free_slot[kMaxCompacted / 2];
  __shared__ int waves[16];
  __shared__ int before_count;
  const int t = threadIdx.x;
  const int each = (slots + kPlanThreads - 1) / kPlanThreads;  // consecutive slots a thread
  const int first = min(t * each, slots), last = min(first + each, slots);
  int own = 0;
  for (int i = first; i < last; ++i) own += live[i] != 0 ? 1 : 0;
  int total;
  const int before = sum_before(own, waves, total);
  if (t == 0) {
    *count = total;
    before_count = total;  // where every place before `total` is live
  }
  __syncthreads();
  // The free places before `total`, in order; how many live ones there are.
  int seen = before;
  for (int i = first; i < last; ++i) {
    if (i == total) before_count = seen;
    const bool is = live[i] != 0;
    if (i < total && !is) free_slot[i - seen] = static_cast<uint16_t>(i);
    seen += is ? 1 : 0;
  }
  __syncthreads();
  seen = before;
  const int moves = total - before_count;
  for (int i = first; i < last; ++i) {
    const bool is = live[i] != 0;
    int to = is ? i : -1;
    if (is && i >= total) {
      const int place = seen - before_count;
      to = free_slot[place];
      steps[place] = make_int4(i, to, 0, place + 1);
    }
    placed[i] = to;
    seen += is ? 1 : 0;
  }
  for (int i = moves + t; i < (slots + 1) / 2; i += kPlanThreads) {
    steps[i] = make_int4(-1, -1, 0, i + 1);
  }
}

// ------------------------------------------------------------------- copies

constexpr int kCopyThreads = 256;
// Rows whose loads are all asked for before the first store, by the workgroups that one slot
// takes.  Chains and cycles are one part of the grid each, and their few workgroups wait for
// latency: a cycle of 500 slots takes, with 8 rows and with 1, 45 and 124 us on 8 workgroups
// (32 KiB), 117 and 344 on 128, 212 and 402 on 256, 424 and 467 on 512, 640 and 633 on 768, 856
// and 812 on 1,024 (4 MiB: reads of slots that lie a power of two apart cost more than they
// hide), 300 encoded slots of 32 heads (218) permuted 129 and 214, 96 beams of 2 MiB (512) 60
// and 79.  Forks, whose pairs spread over the grid's second dimension, have less to wait for and
// pay: those encoded slots 52 and 49, 96 slots of 512 KiB (128) 16 and 12, of 2 MiB 38 and 36.
// The rule is the chains', which gain more than forks lose; 96 beams of 8 layers (4,096) take
// 527 and 508.  4 rows are between the two, 16 no faster than 8.
constexpr int kBatchOfFew = 8, kBatchOfMany = 1;
constexpr uint64_t kManyWorkgroups = 4 * kComputeUnits;
constexpr int kFewBuffers = 9;    // of a launch with a small argument block (2 us less of a call)
constexpr int kMostBuffers = 64;  // of one launch
// Workgroups that fill the card: 8, 16, 32 and 64 a compute unit copy the 300 encoded slots in
// 56.9, 56.8, 55.6 and 57.1 us, the 90 of 4 layers in 107, 106, 102 and 105.
constexpr uint32_t kFill = 32 * kComputeUnits;

struct CopyBuffer {
  const char* from;
  char* to;
  uint64_t bytes;       // a slot
  uint32_t first;       // its first workgroup
  uint32_t unit;        // bytes a thread: 16, 4 or 1
};

template <int kMost>
struct CopyArgs {
  CopyBuffer buffers[kMost];
  const int4* steps;
  uint32_t count, rows, slots;
};

// x of one lane.
__device__ __forceinline__ uint64_t lane_value(uint64_t x, int lane) {
  const uint32_t low = __builtin_amdgcn_readlane(static_cast<uint32_t>(x), lane);
  const uint32_t high = __builtin_amdgcn_readlane(static_cast<uint32_t>(x >> 32), lane);
  return static_cast<uint64_t>(high) << 32 | low;
}

// Rows begin .. end - 1 for the threads' runs of `sizeof(Unit)` bytes from byte `start` of
// every slot on.  A wavefront's lanes hold a row of the plan each, 64 at a time, and kBatch of
// them are carried out together: all loads, then all stores, up to a row that writes what was
// kept (so that one value is kept at a time).  A row that reads nothing loads from the first
// slot, so that no load depends on a branch.  Loads are plain: with the nontemporal hint the
// 96 slots above take 557 us and not 519, since rows that read one slot do not share it.
template <typename Unit, int kBatch>
__device__ __forceinline__ void copy_rows(const CopyBuffer& b, uint64_t start, const int4* steps,
                                          uint32_t begin, uint32_t end, uint32_t slots) {
  constexpr uint32_t kAll = (1u << kBatch) - 1;
  const uint32_t offset = threadIdx.x * sizeof(Unit);
  const bool active = start + offset < b.bytes;
  const char* const from = b.from + start;
  char* const to = b.to + start;
  const int lane = threadIdx.x & 63;
  Unit kept = {};
  for (uint32_t chunk = begin; chunk < end; chunk += 64) {
    const bool in = chunk + lane < end;
    const int4 row = steps[in ? chunk + lane : begin];
    const bool writes = in && static_cast<uint32_t>(row.y) < slots;
    const bool reads = writes && static_cast<uint32_t>(row.x) < slots && !(row.z & kSaved);
    const uint64_t target = writes ? row.y * b.bytes : 0, source = reads ? row.x * b.bytes : 0;
    const uint64_t all_write = __ballot(writes), all_read = __ballot(reads);
    const uint64_t all_save = __ballot(writes && (row.z & kSaves));
    const uint64_t all_saved = __ballot(writes && (row.z & kSaved));
    int first = 0;
    while (first < 64 && all_write >> first != 0) {
      const uint32_t saved = static_cast<uint32_t>(all_saved >> first) & kAll;
      const uint32_t some = saved ? (saved ^ (saved - 1)) : kAll;  // up to the lowest
      const uint32_t write = static_cast<uint32_t>(all_write >> first) & some;
      const uint32_t read = static_cast<uint32_t>(all_read >> first) & some;
      const uint32_t save = static_cast<uint32_t>(all_save >> first) & some;
      const char* at[kBatch];
      char* out[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        at[i] = from + lane_value(source, first + i);
        out[i] = to + lane_value(target, first + i);
      }
      const char* const keep = from + lane_value(target, first + __builtin_ctz(save | 1u << 31));
      if (active) {
        Unit x[kBatch];
        if (read) {
#pragma unroll
          for (int i = 0; i < kBatch; ++i) x[i] = *reinterpret_cast<const Unit*>(at[i] + offset);
        }
        if (save) kept = *reinterpret_cast<const Unit*>(keep + offset);
        if ((read & write) == kAll) {
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            __builtin_nontemporal_store(x[i], reinterpret_cast<Unit*>(out[i] + offset));
          }
        } else {
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            if (write >> i & 1) {
              const Unit value = read >> i & 1 ? x[i] : saved >> i & 1 ? kept : Unit{};
              __builtin_nontemporal_store(value, reinterpret_cast<Unit*>(out[i] + offset));
            }
          }
        }
      }
      first += saved ? __builtin_ctz(saved) + 1 : kBatch;
    }
  }
}

// The first row of part `part` of `parts`, moved on to the end of a tree.
__device__ __forceinline__ uint32_t part_begin(const int4* steps, uint32_t rows, uint32_t part,
                                               uint32_t parts) {
  const uint32_t at = static_cast<uint32_t>(static_cast<uint64_t>(rows) * part / parts);
  if (at == 0 || at >= rows) return min(at, rows);
  return min(max(static_cast<uint32_t>(steps[at - 1].w), at), rows);
}

template <int kMost, int kBatch>
__global__ __launch_bounds__(kCopyThreads) void copy_slots_kernel(CopyArgs<kMost> a) {
  uint32_t i = 0;
  while (i + 1 < a.count && a.buffers[i + 1].first <= blockIdx.x) ++i;
  const CopyBuffer b = a.buffers[i];
  const uint32_t begin = part_begin(a.steps, a.rows, blockIdx.y, gridDim.y);
  const uint32_t end = part_begin(a.steps, a.rows, blockIdx.y + 1, gridDim.y);
  const uint64_t at = static_cast<uint64_t>(blockIdx.x - b.first) * kCopyThreads * b.unit;
  if (b.unit == 16) copy_rows<u32x4_t, kBatch>(b, at, a.steps, begin, end, a.slots);
  else if (b.unit == 4) copy_rows<uint32_t, kBatch>(b, at, a.steps, begin, end, a.slots);
  else copy_rows<uint8_t, kBatch>(b, at, a.steps, begin, end, a.slots);
}

// Bytes a thread copies of a slot: what the addresses and sizes of a buffer are multiples of.
uint32_t unit_of(const gdn_state_codec_slot_buffer& b) {
  const uint64_t bits =
      reinterpret_cast<uintptr_t>(b.from) | reinterpret_cast<uintptr_t>(b.to) | b.bytes;
  return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
}
uint64_t workgroups_of(const gdn_state_codec_slot_buffer& b) {
  const uint64_t run = static_cast<uint64_t>(unit_of(b)) * kCopyThreads;
  return (b.bytes + run - 1) / run;
}

template <int kMost>
int32_t launch_copy(void* stream, const gdn_state_codec_slot_buffer* buffers, uint32_t count,
                    const int32_t* steps, uint32_t rows, uint32_t slots) {
  CopyArgs<kMost> args;
  args.steps = reinterpret_cast<const int4*>(steps);
  args.count = count;
  args.rows = rows;
  args.slots = slots;
  uint64_t blocks = 0;
  for (uint32_t i = 0; i < count; ++i) {
    const gdn_state_codec_slot_buffer& b = buffers[i];
    args.buffers[i] = {static_cast<const char*>(b.from), static_cast<char*>(b.to), b.bytes,
                       static_cast<uint32_t>(blocks), unit_of(b)};
    blocks += workgroups_of(b);
  }
  uint64_t parts = (kFill + blocks - 1) / blocks;
  if (parts > rows) parts = rows;
  return launch(blocks < kManyWorkgroups ? copy_slots_kernel<kMost, kBatchOfFew>
                                         : copy_slots_kernel<kMost, kBatchOfMany>,
                dim3(static_cast<uint32_t>(blocks), static_cast<uint32_t>(parts)),
                dim3(kCopyThreads), stream, args);
}

}  // namespace
}  // namespace gdn

extern "C" int32_t statecentric_gdn_state_codec_slot_moves_launch_v1(
    void* stream, const int32_t* sources, const int32_t* targets, uint32_t pairs, uint32_t slots,
    int32_t* steps) {
  if (!sources || !targets || !steps || pairs == 0 || pairs > GDN_STATE_CODEC_MAX_MOVES ||
      slots == 0 || slots > 0x7FFFFFFFu || !gdn::aligned16(sources, targets, steps)) {
    return gdn::kStatusInvalidArgument;
  }
  uint32_t table = 2, threads = 64;
  while (table < 2 * pairs) table *= 2;
  while (threads < pairs && threads < gdn::kPlanThreads) threads *= 2;
  return gdn::launch(gdn::slot_moves_kernel, dim3(1), dim3(threads), stream, sources, targets,
                     static_cast<int>(pairs), slots, table, reinterpret_cast<int4*>(steps));
}

extern "C" int32_t statecentric_gdn_state_codec_compaction_moves_launch_v1(
    void* stream, const int32_t* live, uint32_t slots, int32_t* steps, int32_t* placed,
    int32_t* count) {
  if (!live || !steps || !placed || !count || slots == 0 ||
      slots > GDN_STATE_CODEC_MAX_COMPACTED || !gdn::aligned16(live, steps, placed, count)) {
    return gdn::kStatusInvalidArgument;
  }
  return gdn::launch(gdn::compaction_kernel, dim3(1), dim3(gdn::kPlanThreads), stream, live,
                     static_cast<int>(slots), reinterpret_cast<int4*>(steps), placed, count);
}

extern "C" int32_t statecentric_gdn_state_codec_copy_slots_launch_v1(
    void* stream, const gdn_state_codec_slot_buffer* buffers, uint32_t count,
    const int32_t* steps, uint32_t rows, uint32_t slots) {
  if (!buffers || !steps || count == 0 || rows == 0 || rows > 0x7FFFFFFFu || slots == 0 ||
      slots > 0x7FFFFFFFu || !gdn::aligned16(steps)) {
    return gdn::kStatusInvalidArgument;
  }
  // Every buffer's size fits an address, and every launch's threads its grid.
  uint64_t blocks = 0;
  for (uint32_t i = 0; i < count; ++i) {
    const uint64_t bytes = buffers[i].bytes;
    if (!buffers[i].from || !buffers[i].to || bytes == 0 || bytes > (1ull << 47) / slots) {
      return gdn::kStatusInvalidArgument;
    }
    if (i % gdn::kMostBuffers == 0) blocks = 0;
    blocks += gdn::workgroups_of(buffers[i]);
    if (blocks > gdn::kMaxGrid / gdn::kCopyThreads) return gdn::kStatusInvalidArgument;
  }
  for (uint32_t done = 0; done < count; done += gdn::kMostBuffers) {
    const uint32_t some = count - done < gdn::kMostBuffers ? count - done : gdn::kMostBuffers;
    const int32_t status =
        some <= gdn::kFewBuffers
            ? gdn::launch_copy<gdn::kFewBuffers>(stream, buffers + done, some, steps, rows, slots)
            : gdn::launch_copy<gdn::kMostBuffers>(stream, buffers + done, some, steps, rows,
                                                  slots);
    if (status != gdn::kStatusOk) return status;
  }
  return gdn::kStatusOk;
}
