// The sequential half of the gated delta rule's chunked form, forward
// (formulas, layouts and precision in delta_chunk.h).
//
// Column v of a state [key][value] meets only column v of V, E and O, so columns
// go to wavefronts and workgroups as they like, but from S0 to S1 is one chain,
//   S0 -> K S0 -> R -> (N b) R -> E -> K^T U -> S1,
// chunk after chunk.  Per chunk and 16 columns it issues
//   K S0: 48, (N b) R: 36, K^T U: 48, and beside the chain Q S0: 32, (P b) E: 18
// matrix instructions.  Two forms, and a third made of the first:
//
// delta_scan_wide_kernel, for throughput: a workgroup takes 64 columns, with two
// wavefronts for each 16.  One runs the chain with all 64 tokens, the state in its
// accumulators: what one product hands to the next are accumulators cut into parts, in
// registers, with no exchange.  The other loads the operands, which all share, into LDS
// half a chunk ahead, forms the outputs half a chunk behind and stores what training
// keeps; it takes S0 and E from LDS.  Bound by the chain's 132 matrix instructions and
// the vector instructions between them: 3.1 us a chunk (32 heads of one request), where
// the products alone would take 0.9; in training by the 112 KiB a chunk and head that it
// stores, 5.4 us (128 heads at once, 2.7 TB/s; without the stores 3.8).  With one
// wavefront for both the chain and the rest these were 4.1 and 6.8.
//
// delta_scan_narrow_kernel, for few heads, where a long request's chain is all there
// is: a workgroup takes 16 columns, and its wavefronts share each product by token
// rows (or state rows), four on the chain and four on the outputs.  What a product
// hands to the next goes through LDS, three exchanges a chunk; a wavefront's own
// operands go from global memory to its registers a chunk ahead.  2.1 us a chunk.
//
// delta_segment_kernel, for long requests of few heads: the chain is linear in the state,
// S1 = M S0 + B, so a request's chunks are cut into segments whose B and M (the same
// chain from zeros, and from the identity without values) are found at once; joined in
// order (delta_join_kernel) they give each segment's start, from which a second pass
// runs all segments at once.  About three times the work, on all compute units instead
// of a few.  With unit keys and strengths of 0 to 1 every M is a contraction; with others
// it grows as the states themselves would.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "delta_chunk.h"

namespace gdn {

int32_t launch_delta_prepare(void* stream, const RuleArgs& args, bf16_bits* outputs);

struct ScanArgs {
  RuleArgs rule;
  const void* initial;       // states [..][value head][value][key], or null: zeros
  void* final_states;        // may be `initial`
  const int32_t* slot_ids;   // of each request, or null: the request's own place
  const int32_t* resume;     // 0: start from zeros, or null: all resume
  uint32_t slots;
  bf16_bits* outputs;        // [tokens][value head][128]
  uint32_t segments;         // after a request's first, and which of the two passes
  uint32_t pass;
};

namespace {

// Where one workgroup works: a request's value head, and its tokens and chunk rows as
// far as the tables stay inside the batch.
struct Work {
  uint32_t head, request;
  uint64_t tile;  // of the state
  uint32_t first_row, begin, length, chunks;
  bool resumed;
};

// Item `item` of requests x value heads, longest requests first; false: none, or
// padding.
__device__ __forceinline__ bool find_work(const ScanArgs& args, uint64_t item, Work& w) {
  const RuleArgs& a = args.rule;
  const ChunkSpace& space = a.space;
  if (item >= static_cast<uint64_t>(a.requests) * space.value_heads) return false;
  w.head = static_cast<uint32_t>(item % space.value_heads);
  w.request = static_cast<uint32_t>(a.order[item / space.value_heads]);
  if (w.request >= a.requests) return false;
  const uint32_t slot =
      args.slot_ids ? static_cast<uint32_t>(args.slot_ids[w.request]) : w.request;
  if (slot >= args.slots) return false;
  w.tile = (static_cast<uint64_t>(slot) * space.value_heads + w.head) * kTile;
  w.resumed = args.initial && (!args.resume || args.resume[w.request] != 0);
  w.first_row = min(static_cast<uint32_t>(a.chunk_offsets[w.request]), space.rows);
  const uint32_t rows =
      min(static_cast<uint32_t>(a.chunk_offsets[w.request + 1]), space.rows) - w.first_row;
  w.begin = min(static_cast<uint32_t>(a.offsets[w.request]), a.tokens);
  w.length = min(static_cast<uint32_t>(a.offsets[w.request + 1]), a.tokens) - w.begin;
  w.chunks = min(rows, (w.length + kChunk - 1) / kChunk);
  return true;
}

// One segment of a request's chunks, and what becomes of its state.
struct Segment {
  const float* start;  // the state before it, as accumulators; or null: the pool's, or zeros
  float* end;          // the state after it; or null: the pool's
  bool map;            // from the identity, without values: end = map x start + the rest
  bool outputs, keep;  // whether it forms outputs, and leaves its state
};

// The segments' states of an item: before segments 1.., then the maps of 1.. .
__device__ __forceinline__ float* segment_state(const ScanArgs& args, uint64_t item,
                                                uint32_t at) {
  return args.rule.space.segments() + (item * (2 * args.segments - 1) + at) * kTile;
}

// Task `task` of a pass: `segments` + 1 parts of each item's chunks.  The first pass runs
// the first part whole, and of all others but the last finds what they add (from zeros)
// and, `second`, their maps; the second pass runs all others whole.  The first part is as
// much longer as a chunk of both takes longer than a chunk whole.
__device__ __forceinline__ bool find_segment(const ScanArgs& args, uint64_t task, bool second,
                                             Work& w, Segment& s) {
  const uint64_t items = static_cast<uint64_t>(args.rule.requests) * args.rule.space.value_heads;
  const uint64_t item = task % items;
  const uint32_t n = args.segments;
  const uint32_t part = static_cast<uint32_t>(task / items) + args.pass;
  if (part >= n + args.pass || !find_work(args, item, w)) return false;
  const uint32_t whole = w.chunks;
  const uint32_t first = whole < 4 * n ? whole : (3 * whole + 2 * n + 2) / (2 * n + 3);
  const uint32_t each = (whole - first + n - 1) / n;
  const uint32_t from = part == 0 ? 0 : min(first + (part - 1) * each, whole);
  const uint32_t to = part == 0 ? first : min(from + each, whole);
  s.outputs = part == 0 || args.pass != 0;
  s.map = !s.outputs && second;
  s.start = part == 0 || args.pass == 0 ? nullptr : segment_state(args, item, part - 1);
  s.end = s.map ? segment_state(args, item, n + part - 1)
          : part == n ? nullptr : segment_state(args, item, part);
  s.keep = args.pass == 0 || part == n;
  if (part != 0) w.resumed = false;
  w.first_row += from;
  w.begin += from * kChunk;
  w.length = to == whole ? w.length - from * kChunk : (to - from) * kChunk;
  w.chunks = to - from;
  return true;
}

// A head's state in a wavefront's accumulators: tiles `first`.. of column `value`
// (row 4 g + i of a tile is key state_key).
template <int kTiles, typename Pool>
__device__ __forceinline__ void load_state(const Pool* state, int first, int value, int g,
                                           bool resumed, f32x4 (&x)[kTiles]) {
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    x[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (resumed) x[t] = load_cells(state + value * kDim + state_key(first + t, 4 * g));
  }
}
template <int kTiles, typename Pool>
__device__ __forceinline__ void store_state(Pool* state, int first, int value, int g,
                                            const f32x4 (&x)[kTiles]) {
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    store_cells(state + value * kDim + state_key(first + t, 4 * g), x[t]);
  }
}

// bf16 rows of a tile's four accumulator rows, as a quad of lanes stores them.
__device__ __forceinline__ uint2 output_run(const f32x4& x, int lane) {
  return transpose_quad(make_uint2(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3])), lane);
}
__device__ __forceinline__ f32x4 value_rows(const uint2& run, int lane) {
  const uint2 x = transpose_quad(run, lane);
  return f32x4{widen_low(x.x), widen_high(x.x), widen_low(x.y), widen_high(x.y)};
}

// ------------------------------------------------------------ 64 columns

constexpr int kWideWaves = 4;
constexpr int kWideSlices = kDim / (16 * kWideWaves);

// A chunk's operands in LDS, in two halves, each fetched while the other is at work:
// the factors, N b (20 KiB of the value head's block) and K rows (16 tiles), then Q rows,
// K^T and P b (two stages: it is read a phase later).  Beside them S0 and E (two stages)
// as the chain's accumulators hold them.  156 KiB: a workgroup has the compute unit to
// itself.
constexpr int kBlockTiles = 20;
constexpr int kStageKeys = kBlockTiles * kTileBytes;
constexpr int kStageQueries = kStageKeys + kKeyTiles * kTileBytes;
constexpr int kStageColumns = kStageQueries + kKeyTiles * kTileBytes;
constexpr int kStageRead = kStageColumns + kKeyTiles * kTileBytes;
constexpr int kStageState = kStageRead + 2 * kReadOutBytes;
constexpr int kStageErrors = kStageState + kWideWaves * 8 * kTileBytes;
constexpr int kStage = kStageErrors + 2 * kWideWaves * 4 * kTileBytes;
static_assert(kReadOut <= kBlockTiles * kTileBytes, "factors and N");
static_assert(kStage <= 160 * 1024, "a compute unit's LDS");

// Two bf16 parts of 8 places: 2^-15 of terms whose sums become bf16 outputs.
__device__ __forceinline__ void split2(const f32x4& x, const f32x4& y, uint4 (&part)[2]) {
  uint4 all[3];
  split3(x, y, all);
  part[0] = all[0], part[1] = all[1];
}

// The chain's three products, of one wavefront's 16 columns.  R = V - exp(G) K S0, from
// the state's parts, and from rows of V as fetched (columns 4 (r / 4).. of tokens 16 t +
// 4 g + (r & 3)) or none.
__device__ __forceinline__ void chain_rest(const uint4* const (&k_rows)[4],
                                           const uint4 (&parts)[4][3],
                                           const f32x4 (&factors)[4], const uint2 (&values)[4],
                                           bool none, int lane, f32x4 (&error)[4]) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    f32x4 seen[2] = {};  // two sums, so that each product waits for the last but one
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const uint4 k = k_rows[step][256 * t];
#pragma unroll
      for (int p = 2; p >= 0; --p) seen[p & 1] = mfma(k, parts[step][p], seen[p & 1]);
    }
    const f32x4 read_key = of_rows(factors[t][kReadKey]);
    f32x4 x = value_rows(values[t], lane);
    if (none) x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) error[t][i] = fmaf(-read_key[i], seen[0][i] + seen[1][i], x[i]);
  }
}

// E = R + (N b) R
__device__ __forceinline__ void chain_solve(const uint4* solve, f32x4 (&error)[4]) {
  uint4 part[2][3];
#pragma unroll
  for (int step = 0; step < 2; ++step) {
    split3(error[2 * step], error[2 * step + 1], part[step]);
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int step = 0; step < lower_steps(t); ++step) {
      uint4 n[3];
#pragma unroll
      for (int p = 0; p < 3; ++p) n[p] = solve[(p * kTriangle + lower_tile(t, step)) * 64];
      error[t] = mfma6(n, part[step], error[t]);
    }
  }
}

// S1 = exp(G_63) S0 + K^T (write b E)
__device__ __forceinline__ void chain_state(const uint4* k_columns, const f32x4 (&factors)[4],
                                            const f32x4 (&error)[4], f32x4 (&state)[8]) {
#pragma unroll
  for (int t = 0; t < 8; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) state[t][i] *= factors[0][kWhole];
  }
#pragma unroll
  for (int step = 0; step < 2; ++step) {
    uint4 written[3];
    f32x4 x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const f32x4 write = of_rows(factors[2 * step + u][kWrite]);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[u][i] = write[i] * error[2 * step + u][i];
    }
    split3(x[0], x[1], written);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      state[t] = mfma3(k_columns[(2 * t + step) * 64], written, state[t]);
    }
  }
}

// A request's chunks, or one segment's, of the value head and columns `block` of `w`.
template <typename Pool, bool kTrain, bool kSplit>
__device__ __forceinline__ void scan_columns(const ScanArgs& args, const Work& w,
                                             const Segment& part, int block, char* stage) {
  const RuleArgs& a = args.rule;
  const ChunkSpace& space = a.space;
  const int place = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = place % kWideWaves;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int slice = kWideWaves * block + wave;
  const int first_value = 16 * slice, value = first_value + r;
  const uint32_t key_head = w.head / a.group;
  const uint32_t length = w.length, chunks = w.chunks;
  f32x4* const state_cells =
      reinterpret_cast<f32x4*>(stage + kStageState) + wave * 8 * 64 + lane;
  const auto error_cells = [&](uint32_t c) {
    return reinterpret_cast<f32x4*>(stage + kStageErrors) +
           ((c & 1) * kWideWaves + wave) * 4 * 64 + lane;
  };

  if (place >= kWideWaves) {  // the operands' loads, the outputs, training's stores
    const uint32_t stage_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) char*)stage));
    const uint32_t key_step = static_cast<uint32_t>(a.key_stride) * 2;
    const uint32_t query_step = static_cast<uint32_t>(a.query_stride) * 2;
    const uint32_t out_step = space.value_heads * kDim * 2;
    const uint32_t linear = 16 * lane;
    const auto fetch_first = [&](uint32_t c) {
      const uint64_t token = w.begin + c * kChunk;
      const uint32_t last = min(length - c * kChunk, static_cast<uint32_t>(kChunk)) - 1;
      const char* k = reinterpret_cast<const char*>(a.keys + token * a.key_stride +
                                                    key_head * kDim);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        stage_rows(k, key_step, last, kWideWaves * i + wave, lane, stage_at + kStageKeys);
      }
      const char* block = space.value_block(w.first_row + c, w.head);
#pragma unroll
      for (int i = 0; i < kBlockTiles / kWideWaves; ++i) {
        const int tile = kWideWaves * i + wave;
        stage_tile(block + tile * kTileBytes, linear, stage_at + tile * kTileBytes);
      }
    };
    const auto fetch_second = [&](uint32_t c) {
      const uint64_t token = w.begin + c * kChunk;
      const uint32_t last = min(length - c * kChunk, static_cast<uint32_t>(kChunk)) - 1;
      const char* columns = space.key_block(w.first_row + c, key_head) + kKeyColumns;
      const char* q = reinterpret_cast<const char*>(a.queries + token * a.query_stride +
                                                    key_head * kDim);
      const char* read = space.value_block(w.first_row + c, w.head) + kReadOut;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tile = kWideWaves * i + wave;
        stage_tile(columns + tile * kTileBytes, linear,
                   stage_at + kStageColumns + tile * kTileBytes);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        stage_rows(q, query_step, last, kWideWaves * i + wave, lane, stage_at + kStageQueries);
      }
#pragma unroll
      for (int i = 0; i < 2 * kTriangle / kWideWaves; ++i) {
        const int tile = kWideWaves * i + wave;
        stage_tile(read + tile * kTileBytes, linear,
                   stage_at + kStageRead + (c & 1) * kReadOutBytes + tile * kTileBytes);
      }
    };
    f32x4 out[4], error[4];
    uint2 runs[4];
    const auto read_errors = [&](uint32_t c) {  // O += (P b) E, and both as they are stored
      const f32x4* const cells = error_cells(c);
      const uint4* const read_out =
          reinterpret_cast<const uint4*>(stage + kStageRead + (c & 1) * kReadOutBytes) + lane;
#pragma unroll
      for (int t = 0; t < 4; ++t) error[t] = cells[64 * t];
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        uint4 part[2];
        split2(error[2 * step], error[2 * step + 1], part);
#pragma unroll
        for (int t = 2 * step; t < 4; ++t) {  // rows 0..31 end in step 0
          const int tile = lower_tile(t, step);
          const uint4 high = read_out[tile * 64], low = read_out[(kTriangle + tile) * 64];
          out[t] = mfma(low, part[0], out[t]);
          out[t] = mfma(high, part[1], out[t]);
          out[t] = mfma(high, part[0], out[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        runs[t] = output_run(out[t], lane);
        if constexpr (kTrain) error[t] = transpose_quad(error[t], lane);
      }
    };
    // kTrain ? 8 : 4 stores, of which the tokens past `tokens` have none.
    const auto store_rows = [&](uint32_t c, int tokens) {
      char* o = reinterpret_cast<char*>(args.outputs) +
                (w.begin + static_cast<uint64_t>(c) * kChunk) * out_step +
                2 * (w.head * kDim + first_value);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int token = 16 * t + 4 * g + (r & 3);
        if (token < tokens) store_run(o, token * out_step + 2 * (r & 12), runs[t]);
        if constexpr (kTrain) {
          store_run(space.errors(w.first_row + c, w.head) + slice * slice_cells(4),
                    t * kTileBytes + linear, error[t]);
        }
      }
    };
    const uint4* q_rows[4];
    row_operands(stage + kStageQueries, lane, q_rows);
    if (chunks != 0) fetch_first(0);
    for (uint32_t c = 0; c < chunks; ++c) {
      // The first half is there, the second has been read.  Only the stores issued after
      // the tiles stay in flight: a store's way to memory is as long as a chunk's work.
      if (c < 2) {
        stage_ready();
      } else {
        stage_ready<kTrain ? 8 : 4>();
      }
      fetch_second(c);
      f32x4 state[8];
      float queries[4];
#pragma unroll
      for (int t = 0; t < 8; ++t) state[t] = state_cells[64 * t];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        queries[t] =
            reinterpret_cast<const float*>(stage)[kReadQuery + 16 * t + 4 * g + (r & 3)];
      }
      uint4 parts[4][2];
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        split2(state[2 * step], state[2 * step + 1], parts[step]);
      }
      if constexpr (kTrain) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          store_run(space.state(w.first_row + c, w.head) + slice * slice_cells(8),
                    t * kTileBytes + linear, transpose_quad(state[t], lane));
        }
      }
      if (c != 0) read_errors(c - 1);
      // The second half and E are there, the first half and S0 have been read.
      stage_ready<kTrain ? 8 : 0>();
      if (c + 1 < chunks) fetch_first(c + 1);
      if (c != 0) store_rows(c - 1, kChunk);  // only the last chunk can be short
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 read[2] = {};
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          const uint4 q = q_rows[step][256 * t];
          read[0] = mfma(q, parts[step][1], read[0]);
          read[1] = mfma(q, parts[step][0], read[1]);
        }
        const f32x4 read_query = of_rows(queries[t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) out[t][i] = read_query[i] * (read[0][i] + read[1][i]);
      }
    }
    if (chunks != 0) {
      read_errors(chunks - 1);
      store_rows(chunks - 1, length - (chunks - 1) * kChunk);
    }
    return;
  }

  // The chain.
  f32x4 state[8];
  if (kSplit && part.start) {
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      state[t] = load4(part.start + slice * slice_cells(8) + 256 * t + 4 * lane);
    }
  } else {
    load_state(static_cast<const Pool*>(args.initial) + w.tile, 0, value, g, w.resumed, state);
  }
  const uint32_t value_step = static_cast<uint32_t>(a.value_stride) * 2;
  uint2 values[4];  // columns 4 (r / 4).. of tokens 16 t + 4 g + (r & 3)
  const auto fetch_values = [&](uint32_t c) {
    const uint64_t token = w.begin + c * kChunk;
    const uint32_t last = min(length - c * kChunk, static_cast<uint32_t>(kChunk)) - 1;
    const char* v = reinterpret_cast<const char*>(a.values + token * a.value_stride +
                                                  w.head * kDim + first_value);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t row = min(static_cast<uint32_t>(16 * t + 4 * g + (r & 3)), last);
      values[t] = *reinterpret_cast<const uint2*>(v + (row * value_step + 2 * (r & 12)));
    }
  };
  const uint4* k_rows[4];
  row_operands(stage + kStageKeys, lane, k_rows);
  const uint4* const k_columns = reinterpret_cast<const uint4*>(stage + kStageColumns) + lane;
  const uint4* const solve = reinterpret_cast<const uint4*>(stage + kSolve) + lane;
  if (chunks != 0) fetch_values(0);
  for (uint32_t c = 0; c < chunks; ++c) {
    uint4 parts[4][3];  // of the state, over the keys
#pragma unroll
    for (int t = 0; t < 8; ++t) state_cells[64 * t] = state[t];
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      split3(state[2 * step], state[2 * step + 1], parts[step]);
    }
    exchange();
    f32x4 factors[4];  // of tokens 16 t + 4 g + (r & 3)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      factors[t] = reinterpret_cast<const f32x4*>(stage)[16 * t + 4 * g + (r & 3)];
    }
    f32x4 error[4];
    chain_rest(k_rows, parts, factors, values, false, lane, error);
    if (c + 1 < chunks) fetch_values(c + 1);
    chain_solve(solve, error);
    f32x4* const cells = error_cells(c);
#pragma unroll
    for (int t = 0; t < 4; ++t) cells[64 * t] = error[t];
    exchange();
    chain_state(k_columns, factors, error, state);
  }
  if (kSplit && !part.keep) return;
  if (kSplit && part.end) {
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      store_cells(part.end + slice * slice_cells(8) + 256 * t + 4 * lane, state[t]);
    }
  } else {
    store_state(static_cast<Pool*>(args.final_states) + w.tile, 0, value, g, state);
  }
}

template <typename Pool, bool kTrain>
__global__ __launch_bounds__(128 * kWideWaves) void delta_scan_wide_kernel(ScanArgs args) {
  __shared__ __align__(16) char stage[kStage];
  // A head's slices share their operands: they get consecutive places of one XCD
  // (the dispatcher deals workgroups out to the 8 XCDs in turn).
  const uint32_t turn = blockIdx.x >> 3;
  Work w;
  if (!find_work(args, static_cast<uint64_t>(turn / kWideSlices) * 8 + (blockIdx.x & 7), w)) {
    return;
  }
  scan_columns<Pool, kTrain, false>(args, w, Segment{}, turn % kWideSlices, stage);
}

// ------------------------------------------------------------ segments

// What a segment makes of its state and no more: eight wavefronts, all columns, each the
// chain of 16.  The factors, N b, K rows and K^T of a chunk come into LDS while the last
// chunk is at work.
constexpr int kChainKeys = kBlockTiles * kTileBytes;
constexpr int kChainColumns = kChainKeys + kKeyTiles * kTileBytes;
constexpr int kChainStage = kChainColumns + kKeyTiles * kTileBytes;
static_assert(2 * kChainStage <= kStage, "two stages in the other form's LDS");

__device__ __forceinline__ void scan_state(const ScanArgs& args, const Work& w,
                                           const Segment& part, char* stage) {
  constexpr int kWaves = 8;
  const RuleArgs& a = args.rule;
  const ChunkSpace& space = a.space;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int value = 16 * wave + r;
  const uint32_t key_head = w.head / a.group;
  const uint32_t length = w.length, chunks = w.chunks;
  const uint32_t stage_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) char*)stage));
  const uint32_t key_step = static_cast<uint32_t>(a.key_stride) * 2;
  const uint32_t value_step = static_cast<uint32_t>(a.value_stride) * 2;
  const uint32_t linear = 16 * lane;
  uint2 values[4];
  // Piece i of 0..6; and the values.
  const auto fetch = [&](uint32_t c, int i) {
    const uint32_t to = stage_at + (c & 1) * kChainStage;
    if (i < 2) {
      const uint64_t token = w.begin + c * kChunk;
      const uint32_t last = min(length - c * kChunk, static_cast<uint32_t>(kChunk)) - 1;
      const char* k = reinterpret_cast<const char*>(a.keys + token * a.key_stride +
                                                    key_head * kDim);
      stage_rows(k, key_step, last, kWaves * i + wave, lane, to + kChainKeys);
    } else if (i < 4) {
      const int tile = kWaves * (i - 2) + wave;
      stage_tile(space.key_block(w.first_row + c, key_head) + kKeyColumns + tile * kTileBytes,
                 linear, to + kChainColumns + tile * kTileBytes);
    } else {
      const int tile = min(kWaves * (i - 4) + wave, kBlockTiles - 1);  // the last one again
      stage_tile(space.value_block(w.first_row + c, w.head) + tile * kTileBytes, linear,
                 to + tile * kTileBytes);
    }
  };
  const auto fetch_values = [&](uint32_t c) {
    const uint64_t token = w.begin + c * kChunk;
    const uint32_t last = min(length - c * kChunk, static_cast<uint32_t>(kChunk)) - 1;
    const char* v = reinterpret_cast<const char*>(a.values + token * a.value_stride +
                                                  w.head * kDim + 16 * wave);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t row = min(static_cast<uint32_t>(16 * t + 4 * g + (r & 3)), last);
      values[t] = *reinterpret_cast<const uint2*>(v + (row * value_step + 2 * (r & 12)));
    }
  };

  f32x4 state[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      state[t][i] = part.map && state_key(t, 4 * g + i) == value ? 1.0f : 0.0f;
    }
  }
  if (chunks != 0) {
#pragma unroll
    for (int i = 0; i < 7; ++i) fetch(0, i);
    fetch_values(0);
  }
  for (uint32_t c = 0; c < chunks; ++c) {
    stage_ready();  // this chunk's operands are there, the last one's have been read
    const char* const at = stage + (c & 1) * kChainStage;
    const uint32_t next = min(c + 1, chunks - 1);
    f32x4 factors[4];  // of tokens 16 t + 4 g + (r & 3)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      factors[t] = reinterpret_cast<const f32x4*>(at)[16 * t + 4 * g + (r & 3)];
      // Used before the next loads are issued, so that no wait for it covers them.
      asm volatile("" : "+v"(values[t].x), "+v"(values[t].y));
    }
    uint4 parts[4][3];  // of the state, over the keys
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      split3(state[2 * step], state[2 * step + 1], parts[step]);
      __builtin_amdgcn_sched_barrier(0);
      if (c + 1 < chunks) {
        fetch(c + 1, 2 * step);
        if (step < 3) fetch(c + 1, 2 * step + 1);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    f32x4 error[4];
    const uint4* k_rows[4];
    row_operands(at + kChainKeys, lane, k_rows);
    chain_rest(k_rows, parts, factors, values, part.map, lane, error);
    fetch_values(next);
    chain_solve(reinterpret_cast<const uint4*>(at + kSolve) + lane, error);
    chain_state(reinterpret_cast<const uint4*>(at + kChainColumns) + lane, factors, error,
                state);
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    store_cells(part.end + wave * slice_cells(8) + 256 * t + 4 * lane,
                part.map ? transpose_quad(state[t], lane) : state[t]);
  }
}

template <typename Pool>
__global__ __launch_bounds__(128 * kWideWaves) void delta_segment_kernel(ScanArgs args) {
  __shared__ __align__(16) char stage[kStage];
  const uint32_t turn = blockIdx.x >> 3;  // the two workgroups of a segment on one XCD
  const uint64_t task = static_cast<uint64_t>(turn / 2) * 8 + (blockIdx.x & 7);
  Work w;
  Segment part;
  if (!find_segment(args, task, turn % 2 != 0, w, part)) return;
  if (part.outputs) {
    scan_columns<Pool, false, true>(args, w, part, turn % 2, stage);
  } else {
    scan_state(args, w, part, stage);
  }
}

// The states before segments 2..: a segment's map times the state before it, and what it
// adds (which its place holds).  One workgroup per item and 16 columns, wavefront w the
// state's tiles 2 w and 2 w + 1.
__global__ __launch_bounds__(256) void delta_join_kernel(ScanArgs args) {
  __shared__ uint4 parts[4][3][64];
  const uint64_t item = blockIdx.x / 8;
  Work w;
  if (!find_work(args, item, w)) return;
  const int slice = blockIdx.x % 8;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const uint32_t n = args.segments;
  const int at = slice * slice_cells(8) + 2 * wave * 256 + 4 * lane;
  f32x4 state[2], map[2][4][2], more[2];
  const auto fetch = [&](uint32_t part) {  // for the state after segment `part`
    const float* m = segment_state(args, item, n + part - 1);
    const float* rest = segment_state(args, item, part) + at;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      more[u] = load4(rest + 256 * u);
      const float* p = m + cells_at(8, 2 * wave + u, r, g);
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        map[u][step][0] = load4(p + 2 * step * slice_cells(8));
        map[u][step][1] = load4(p + 2 * step * slice_cells(8) + 16);
      }
    }
  };
#pragma unroll
  for (int u = 0; u < 2; ++u) state[u] = load4(segment_state(args, item, 0) + at + 256 * u);
  fetch(1);
  for (uint32_t part = 1; part < n; ++part) {
    uint4 own[3], factor[2][4][3];
    split3(state[0], state[1], own);
#pragma unroll
    for (int p = 0; p < 3; ++p) parts[wave][p][lane] = own[p];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      state[u] = more[u];
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        split3(map[u][step][0], map[u][step][1], factor[u][step]);
      }
    }
    fetch(min(part + 1, n - 1));
    exchange();
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const uint4 x[3] = {parts[step][0][lane], parts[step][1][lane], parts[step][2][lane]};
#pragma unroll
      for (int u = 0; u < 2; ++u) state[u] = mfma6(factor[u][step], x, state[u]);
    }
    float* const to = segment_state(args, item, part) + at;
#pragma unroll
    for (int u = 0; u < 2; ++u) store_cells(to + 256 * u, state[u]);
    exchange();  // the parts have been read
  }
}

// ------------------------------------------------------------ 16 columns

template <typename Pool, bool kTrain>
__global__ __launch_bounds__(512) void delta_scan_narrow_kernel(ScanArgs args) {
  constexpr int kSlices = kDim / 16;
  // Parts of S0 (4 steps over the keys), R, write b E and E (2 steps over the
  // tokens).
  __shared__ uint4 state_parts[4][3][64];
  __shared__ uint4 row_parts[2][3][64];
  __shared__ uint4 written_parts[2][3][64];
  __shared__ uint4 error_parts[2][2][64];
  const RuleArgs& a = args.rule;
  const ChunkSpace& space = a.space;
  // A head's slices share their operands: they get consecutive places of one XCD
  // (the dispatcher deals workgroups out to the 8 XCDs in turn).
  const uint32_t turn = blockIdx.x >> 3;
  Work w;
  if (!find_work(args, static_cast<uint64_t>(turn / kSlices) * 8 + (blockIdx.x & 7), w)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int rows = wave & 3;           // this wavefront's token rows, 16 rows..
  const int steps = lower_steps(rows);
  const int slice = turn % kSlices, first_value = 16 * slice, value = first_value + r;
  const uint32_t key_head = w.head / a.group;
  const uint32_t length = w.length, chunks = w.chunks;
  const uint32_t mine = 16 * rows + 4 * g + (r & 3);  // the token whose factors it loads

  // Addresses as in the wide form; past the last chunk, the same again.
  uint64_t token = w.begin;
  uint32_t row = w.first_row;
  uint32_t last = min(length, static_cast<uint32_t>(kChunk)) - 1;
  const auto advance = [&](uint32_t c) {  // to chunk c + 1, if there is one
    const uint32_t on = c + 1 < chunks ? 1 : 0;
    token += on * kChunk;
    row += on;
    last = min(length - (c + on) * kChunk, static_cast<uint32_t>(kChunk)) - 1;
  };

  if (wave >= 4) {  // the outputs: O = exp(G) Q S0 + (P b) E
    const uint32_t query_step = static_cast<uint32_t>(a.query_stride) * 2;
    const uint32_t out_step = space.value_heads * kDim * 2;
    uint4 q_rows[4], read_out[2][2];
    float query;
    const auto fetch_queries = [&]() {
      const char* q = reinterpret_cast<const char*>(a.queries + token * a.query_stride +
                                                    key_head * kDim);
      const uint32_t at = min(static_cast<uint32_t>(16 * rows + r), last) * query_step + 16 * g;
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        q_rows[step] = *reinterpret_cast<const uint4*>(q + 64 * step + at);
      }
      query = reinterpret_cast<const float*>(space.value_block(row, w.head))[kReadQuery + mine];
    };
    const auto fetch_read_out = [&]() {
      const uint4* p =
          reinterpret_cast<const uint4*>(space.value_block(row, w.head) + kReadOut);
#pragma unroll
      for (int step = 0; step < 2; ++step) {  // rows 0..31 have no second step
        const int tile = lower_tile(rows, step < steps ? step : 0);
#pragma unroll
        for (int u = 0; u < 2; ++u) read_out[u][step] = p[(u * kTriangle + tile) * 64 + lane];
      }
    };
    if (chunks != 0) fetch_queries();
    for (uint32_t c = 0; c < chunks; ++c) {
      char* const o = reinterpret_cast<char*>(args.outputs) + token * out_step +
                      2 * (w.head * kDim + first_value);
      const uint32_t live = last;
      exchange();
      fetch_read_out();
      advance(c);
      exchange();  // S0's parts stay until the third
      uint4 part[4][2];
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        part[step][0] = state_parts[step][0][lane];
        part[step][1] = state_parts[step][1][lane];
      }
      __builtin_amdgcn_sched_barrier(0);
      // From two of the state's parts: 2^-15 of terms whose sums become bf16 outputs.
      f32x4 read[2] = {};
#pragma unroll
      for (int p = 1; p >= 0; --p) {
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          read[step & 1] = mfma(q_rows[step], part[step][p], read[step & 1]);
        }
      }
      const f32x4 read_query = of_rows(query);
      f32x4 out;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = read_query[i] * (read[0][i] + read[1][i]);
      exchange();
      uint4 part_e[2][2];
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        part_e[step][0] = error_parts[step][0][lane];
        part_e[step][1] = error_parts[step][1][lane];
      }
      __builtin_amdgcn_sched_barrier(0);
      fetch_queries();
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        if (step < steps) {
          out = mfma(read_out[1][step], part_e[step][0], out);
          out = mfma(read_out[0][step], part_e[step][1], out);
          out = mfma(read_out[0][step], part_e[step][0], out);
        }
      }
      const uint2 x = output_run(out, lane);
      if (mine <= live) *reinterpret_cast<uint2*>(o + (mine * out_step + 2 * (r & 12))) = x;
    }
    return;
  }

  // The chain: token rows 16 wave.., state tiles 2 wave and 2 wave + 1.
  f32x4 state[2];
  load_state(static_cast<const Pool*>(args.initial) + w.tile, 2 * wave, value, g, w.resumed,
             state);
  const uint32_t key_step = static_cast<uint32_t>(a.key_stride) * 2;
  const uint32_t value_step = static_cast<uint32_t>(a.value_stride) * 2;
  uint4 k_rows[4], k_columns[2][2], solve[2][3];
  f32x4 factors;
  uint2 values;
  const auto fetch_keys = [&]() {
    const char* k = reinterpret_cast<const char*>(a.keys + token * a.key_stride +
                                                  key_head * kDim);
    const uint32_t at = min(static_cast<uint32_t>(16 * wave + r), last) * key_step + 16 * g;
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      k_rows[step] = *reinterpret_cast<const uint4*>(k + 64 * step + at);
    }
    const char* v = reinterpret_cast<const char*>(a.values + token * a.value_stride +
                                                  w.head * kDim + first_value);
    values = *reinterpret_cast<const uint2*>(v + (min(mine, last) * value_step + 2 * (r & 12)));
  };
  const auto fetch_solve = [&]() {
    const char* const block = space.value_block(row, w.head);
    const uint4* p = reinterpret_cast<const uint4*>(block + kSolve);
    factors = reinterpret_cast<const f32x4*>(block)[mine];
#pragma unroll
    for (int step = 0; step < 2; ++step) {  // rows 0..31 have no second step
      const int tile = lower_tile(wave, step < steps ? step : 0);
#pragma unroll
      for (int u = 0; u < 3; ++u) solve[step][u] = p[(u * kTriangle + tile) * 64 + lane];
    }
  };
  const auto fetch_columns = [&]() {
    const uint4* k =
        reinterpret_cast<const uint4*>(space.key_block(row, key_head) + kKeyColumns);
#pragma unroll
    for (int step = 0; step < 2; ++step) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        k_columns[u][step] = k[(2 * (2 * wave + u) + step) * 64 + lane];
      }
    }
  };
  if (chunks != 0) {
    fetch_keys();
    fetch_solve();
  }

  for (uint32_t c = 0; c < chunks; ++c) {
    {  // S0, cut into parts
      uint4 part[3];
      split3(state[0], state[1], part);
#pragma unroll
      for (int p = 0; p < 3; ++p) state_parts[wave][p][lane] = part[p];
      if constexpr (kTrain) {
        float* p = space.state(row, w.head) + slice * slice_cells(8) + 2 * wave * 256 + 4 * lane;
#pragma unroll
        for (int u = 0; u < 2; ++u) store_cells(p + 256 * u, transpose_quad(state[u], lane));
      }
    }
    float* const e =
        kTrain ? space.errors(row, w.head) + slice * slice_cells(4) + wave * 256 + 4 * lane
               : nullptr;
    exchange();
    // R = V - exp(G) K S0.  An exchange's values are all asked for before the first
    // is used, and the operands two products ahead (of the next chunk, where this one
    // has no more) are asked for while those are on their way: a wavefront's loads
    // go out one every 16 cycles of the compute unit, and nothing behind them moves.
    uint4 part_s[4][3];
#pragma unroll
    for (int p = 2; p >= 0; --p) {
#pragma unroll
      for (int step = 0; step < 4; ++step) part_s[step][p] = state_parts[step][p][lane];
    }
    __builtin_amdgcn_sched_barrier(0);
    fetch_columns();
    advance(c);
    __builtin_amdgcn_sched_barrier(0);
    const f32x4 read_key = of_rows(factors[kReadKey]), write = of_rows(factors[kWrite]);
    const f32x4 v = value_rows(values, lane);
    f32x4 seen[2] = {};  // two sums, so that each product waits for the last but one
#pragma unroll
    for (int p = 2; p >= 0; --p) {
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        seen[step & 1] = mfma(k_rows[step], part_s[step][p], seen[step & 1]);
      }
    }
    f32x4 error, scaled;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      error[i] = fmaf(-read_key[i], seen[0][i] + seen[1][i], v[i]);
    }
    uint2 half[3];
    split3_half(error, half);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      reinterpret_cast<uint2*>(&row_parts[wave >> 1][p][lane])[wave & 1] = half[p];
    }
    exchange();
    // E = R + (N b) R
    uint4 part_r[2][3];
#pragma unroll
    for (int p = 2; p >= 0; --p) {
#pragma unroll
      for (int step = 0; step < 2; ++step) part_r[step][p] = row_parts[step][p][lane];
    }
    __builtin_amdgcn_sched_barrier(0);
    fetch_keys();
    __builtin_amdgcn_sched_barrier(0);
    if (steps == 2) {
      f32x4 more = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int v = 2; v >= 0; --v) {  // parts u and v with u + v <= 2
#pragma unroll
        for (int u = 2 - v; u >= 0; --u) {
          error = mfma(solve[0][u], part_r[0][v], error);
          more = mfma(solve[1][u], part_r[1][v], more);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) error[i] += more[i];
    } else {
      error = mfma6(solve[0], part_r[0], error);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) scaled[i] = write[i] * error[i];
    split3_half(scaled, half);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      reinterpret_cast<uint2*>(&written_parts[wave >> 1][p][lane])[wave & 1] = half[p];
    }
    split3_half(error, half);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      reinterpret_cast<uint2*>(&error_parts[wave >> 1][p][lane])[wave & 1] = half[p];
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) state[t][i] *= factors[kWhole];
    }
    exchange();
    // S1 = exp(G_63) S0 + K^T (write b E)
    uint4 part_w[2][3];
#pragma unroll
    for (int p = 2; p >= 0; --p) {
#pragma unroll
      for (int step = 0; step < 2; ++step) part_w[step][p] = written_parts[step][p][lane];
    }
    __builtin_amdgcn_sched_barrier(0);
    fetch_solve();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int p = 2; p >= 0; --p) {
#pragma unroll
      for (int step = 0; step < 2; ++step) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          state[u] = mfma(k_columns[u][step], part_w[step][p], state[u]);
        }
      }
    }
    if constexpr (kTrain) store_cells(e, transpose_quad(error, lane));
  }
  store_state(static_cast<Pool*>(args.final_states) + w.tile, 2 * wave, value, g, state);
}

template <typename Pool, bool kTrain>
int32_t scan_by_size(void* stream, const ScanArgs& args) {
  const uint64_t items = static_cast<uint64_t>(args.rule.requests) * args.rule.space.value_heads;
  // Where all narrow workgroups run at once, one on each of the 256 compute units, a
  // chunk takes 2.1 us (32 heads of one request), in the wide form 3.1 us.  Twice as many
  // would take two rounds of the one, and one of the other, which issues a quarter of
  // the loads (128 heads, 4 requests in training: 250 us and 172 us).
  const bool narrow = items * (kDim / 16) <= kComputeUnits;
  const uint64_t blocks = (items + 7) / 8 * 8 * (narrow ? kDim / 16 : kWideSlices);
  if (blocks > kMaxGrid) return kStatusInvalidArgument;
  const dim3 grid(static_cast<uint32_t>(blocks));
  return narrow ? launch(delta_scan_narrow_kernel<Pool, kTrain>, grid, dim3(512), stream, args)
                : launch(delta_scan_wide_kernel<Pool, kTrain>, grid, dim3(128 * kWideWaves),
                         stream, args);
}

// One long request, or a few, of few heads: its chunks in segments, the states between
// them from their maps.
template <typename Pool>
int32_t scan_in_segments(void* stream, ScanArgs args) {
  const uint32_t items = args.rule.requests * args.rule.space.value_heads;
  args.segments = std::min(kComputeUnits / kWideSlices / items, kMostSegments);
  const auto run = [&](uint32_t pass) {
    args.pass = pass;
    return launch(delta_segment_kernel<Pool>, dim3((args.segments * items + 7) / 8 * 8 * 2),
                  dim3(128 * kWideWaves), stream, args);
  };
  int32_t status = run(0);
  if (status == kStatusOk) {
    status = launch(delta_join_kernel, dim3(items * 8), dim3(256), stream, args);
  }
  return status == kStatusOk ? run(1) : status;
}

}  // namespace

int32_t launch_delta_scan(void* stream, const ScanArgs& args, uint32_t dtype) {
  if (args.rule.space.train) return scan_by_size<float, true>(stream, args);
  const uint64_t items = static_cast<uint64_t>(args.rule.requests) * args.rule.space.value_heads;
  // In segments, where a request has so many chunks that the two passes, over all compute
  // units, beat the narrow form's one chain: 64 on the average and 4 for each request x
  // head.  32 heads of one request (narrow form in brackets, whole calls): 32,768 tokens
  // 1,000 us (1,240), 8,192 280 (313), 4,096 158 (147).  8 heads: 32,768 tokens 362 (958),
  // 4,096 90 (118).  One head: 4,096 tokens 78 (113).  The average hides one long request
  // among short ones: 32,768 tokens and one more of another request, 32 heads, go through
  // the wide form's one chain in 1,550 us.
  const uint64_t chunks = args.rule.space.rows / args.rule.requests;
  if (items <= kSplitItems && chunks >= std::max<uint64_t>(kSplitChunks, 4 * items)) {
    return dtype == kDtypeF32 ? scan_in_segments<float>(stream, args)
                              : scan_in_segments<bf16_bits>(stream, args);
  }
  return dtype == kDtypeF32 ? scan_by_size<float, false>(stream, args)
                            : scan_by_size<bf16_bits, false>(stream, args);
}

constexpr uint64_t kMaxStride = 1u << 24;  // elements between tokens

// Checks the caller's arguments and fills the kernels'; false: a bad argument.
bool rule_args(const gdn_state_codec_rule* rule, bool train, RuleArgs& a) {
  if (!rule || !rule->offsets || !rule->chunk_offsets || !rule->chunks || !rule->order ||
      !token_rows(rule->tokens, rule->queries, rule->keys, rule->values, rule->log_decay,
                  rule->beta) ||
      !rule->workspace || rule->requests == 0 || rule->requests > GDN_STATE_CODEC_MAX_REQUESTS ||
      rule->tokens > 0x7FFFFFFFu || rule->rows != rule->tokens / kChunk + rule->requests ||
      rule->key_heads == 0 || rule->value_heads == 0 ||
      rule->value_heads % rule->key_heads != 0 || rule->normalize > 1 ||
      // a chunk's rows are addressed with 32-bit byte offsets
      rule->query_stride > kMaxStride || rule->key_stride > kMaxStride ||
      rule->value_stride > kMaxStride || rule->value_heads > kMaxStride / kDim ||
      rule->query_stride % 8 != 0 || rule->key_stride % 8 != 0 || rule->value_stride % 8 != 0 ||
      static_cast<uint64_t>(rule->rows) * rule->value_heads > kMaxGrid ||
      !element_aligned(rule->log_decay, rule->beta) ||
      !aligned16(rule->queries, rule->keys, rule->values, rule->offsets, rule->chunk_offsets,
                 rule->chunks, rule->order, rule->workspace)) {
    return false;
  }
  a = RuleArgs{rule->queries, rule->keys, rule->values, rule->log_decay, rule->beta,
               rule->query_stride, rule->key_stride, rule->value_stride, rule->offsets,
               rule->chunk_offsets, reinterpret_cast<const int4*>(rule->chunks), rule->order,
               rule->requests, rule->tokens, rule->value_heads / rule->key_heads, rule->scale,
               rule->normalize,
               ChunkSpace{static_cast<char*>(rule->workspace), rule->rows, rule->key_heads,
                          rule->value_heads, train}};
  return rule->workspace_bytes >= a.space.total();
}

}  // namespace gdn

extern "C" uint64_t statecentric_gdn_state_codec_gated_delta_workspace_v1(
    uint32_t rows, uint32_t value_heads, uint32_t key_heads, uint32_t train) {
  return gdn::ChunkSpace{nullptr, rows, key_heads, value_heads, train != 0}.total();
}

extern "C" int32_t statecentric_gdn_state_codec_gated_delta_prefill_launch_v1(
    void* stream, const gdn_state_codec_rule* rule, const int32_t* slot_ids,
    const int32_t* resume, void* pool, uint32_t slots, uint32_t pool_dtype, uint16_t* outputs) {
  gdn::ScanArgs args{};
  if (!gdn::rule_args(rule, false, args.rule) || !slot_ids || !pool ||
      !gdn::token_rows(rule->tokens, outputs) || slots == 0 ||
      slots > 0x7FFFFFFFu || pool_dtype > gdn::kDtypeBF16 ||
      !gdn::aligned16(slot_ids, resume, pool, outputs)) {
    return gdn::kStatusInvalidArgument;
  }
  args.initial = pool, args.final_states = pool, args.slot_ids = slot_ids, args.resume = resume;
  args.slots = slots, args.outputs = outputs;
  const int32_t status = gdn::launch_delta_prepare(stream, args.rule, outputs);
  return status != gdn::kStatusOk ? status : gdn::launch_delta_scan(stream, args, pool_dtype);
}

extern "C" int32_t statecentric_gdn_state_codec_gated_delta_forward_launch_v1(
    void* stream, const gdn_state_codec_rule* rule, const float* initial, float* final_states,
    uint16_t* outputs) {
  gdn::ScanArgs args{};
  if (!gdn::rule_args(rule, true, args.rule) || !final_states ||
      !gdn::token_rows(rule->tokens, outputs) ||
      !gdn::aligned16(initial, final_states, outputs)) {
    return gdn::kStatusInvalidArgument;
  }
  args.initial = initial, args.final_states = final_states, args.slots = rule->requests;
  args.outputs = outputs;
  const int32_t status = gdn::launch_delta_prepare(stream, args.rule, outputs);
  return status != gdn::kStatusOk ? status
                                  : gdn::launch_delta_scan(stream, args, gdn::kDtypeF32);
}
