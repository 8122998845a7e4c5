// Gradients of the gated delta rule's chunked form (formulas of the forward pass,
// layouts and precision in delta_chunk.h).
//
// With dS1 the gradient of a chunk's end state, dO of its outputs:
//   V' = P^T dO + exp(G_63 - G) K dS1,   X = V' + N^T (b V'),   Y = b X (= dV),
//   dS0 = exp(G_63) dS1 + (exp(G) Q)^T dO - (exp(G) K)^T Y
// run chunk after chunk, the last first, a column of the state by itself
// (two kernels, the mirrors of the forward scans).  What is left needs no
// order and takes whole rows (delta_gradient_kernel): with U = b E,
//   F_ij = exp(G_i - G_j) dO_i.U_j (j <= i),   H_ij = exp(G_i - G_j) Y_i.U_j (j < i),
//   dq_i = exp(G_i) S0 dO_i + sum_j F_ij k_j
//   dk_i = - exp(G_i) S0 Y_i - sum_j H_ij k_j                     (as it is read)
//          + exp(G_63 - G_i) dS1 U_i + sum_j F_ji q_j - sum_j H_ji k_j  (as it is written)
//   db_i = X_i.E_i
//   dg_t = exp(G_63) <dS1, S0> + sum_(i>=t) exp(G_i) (q_i.S0 dO_i - k_i.S0 Y_i)
//          + sum_(j<t) exp(G_63 - G_j) k_j.dS1 U_j
//          + sum_(j<t<=i) (F_ij q_i.k_j - H_ij k_i.k_j)
// for unit k and scaled unit q; the raw gradients follow through the norms.  A key
// head's gradients are summed over its value heads in registers, in order.
//
// dg_t takes exactly what crosses token t, every term with its exp(g_t).  (q_i.dq_i +
// k_i.dk_i as read - k_i.dk_i as written, summed from t to the chunk's end, is the same,
// but there the pairs on one side of t, and each token's own, cancel: with log decays of
// -12 their rounding was 5% of the gradients.)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "delta_chunk.h"
#include "lane_exchange.h"

namespace gdn {

bool rule_args(const gdn_state_codec_rule* rule, bool train, RuleArgs& a);

namespace {

struct BackArgs {
  RuleArgs rule;
  const bf16_bits* d_outputs;  // [tokens][value head][128]
  const float* d_final;        // [request][value head][value][key], or null: zeros
  float* d_initial;            // the same, or null
  bf16_bits* d_queries;        // [tokens][key head][128]
  bf16_bits* d_keys;
  bf16_bits* d_values;         // [tokens][value head][128]
  float* d_log_decay;          // [tokens][value head]
  bf16_bits* d_beta;
};

// Where one workgroup works: a request's value head, and its tokens and chunk rows as
// far as the tables stay inside the batch.
struct Work {
  uint32_t head, request, first_row, begin, length, chunks;
  uint64_t tile;  // of the state
};

// Item `item` of requests x value heads, longest requests first; false: none.
__device__ __forceinline__ bool find_work(const RuleArgs& a, uint64_t item, Work& w) {
  const ChunkSpace& space = a.space;
  if (item >= static_cast<uint64_t>(a.requests) * space.value_heads) return false;
  w.head = static_cast<uint32_t>(item % space.value_heads);
  w.request = static_cast<uint32_t>(a.order[item / space.value_heads]);
  if (w.request >= a.requests) return false;
  w.tile = (static_cast<uint64_t>(w.request) * space.value_heads + w.head) * kTile;
  w.first_row = min(static_cast<uint32_t>(a.chunk_offsets[w.request]), space.rows);
  const uint32_t rows =
      min(static_cast<uint32_t>(a.chunk_offsets[w.request + 1]), space.rows) - w.first_row;
  w.begin = min(static_cast<uint32_t>(a.offsets[w.request]), a.tokens);
  w.length = min(static_cast<uint32_t>(a.offsets[w.request + 1]), a.tokens) - w.begin;
  w.chunks = min(rows, (w.length + kChunk - 1) / kChunk);
  return true;
}

// The state's gradient in a wavefront's accumulators, tiles `first`.. of column `value`.
template <int kTiles>
__device__ __forceinline__ void load_final(const float* d_final, uint64_t tile, int first,
                                           int value, int g, f32x4 (&x)[kTiles]) {
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    x[t] = d_final ? load4(d_final + tile + value * kDim + state_key(first + t, 4 * g))
                   : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
}
template <int kTiles>
__device__ __forceinline__ void store_initial(float* d_initial, uint64_t tile, int first,
                                              int value, int g, const f32x4 (&x)[kTiles]) {
  if (!d_initial) return;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    store_cells(d_initial + tile + value * kDim + state_key(first + t, 4 * g), x[t]);
  }
}

// ------------------------------------------------------------ 64 columns

// A chunk's operands in LDS, in two halves, each fetched while the other is at work:
// the factors (2 KiB), N^T b, K rows and Q^T; then K^T and the next chunk's P^T and dO.
// Beside them 48 KiB through which the chain and the wavefronts beside it hand each
// other accumulators, each lane to the same lane: dS1 and, once that has been taken,
// (exp(G) Q)^T dO; P^T dO and, once that has been taken, X.
constexpr int kStageSolve = 2 * kTileBytes;
constexpr int kStageKeys = kStageSolve + kTriangleBytes;
constexpr int kStageQueryColumns = kStageKeys + kKeyTiles * kTileBytes;
constexpr int kStageColumns = kStageQueryColumns + kKeyTiles * kTileBytes;
constexpr int kStageRead = kStageColumns + kKeyTiles * kTileBytes;
constexpr int kStageOuts = kStageRead + kTriangleBytes;
constexpr int kWaves = 4;
constexpr int kSlices = kDim / (16 * kWaves);
constexpr int kOutBytes = 32 * kWaves;  // of a token's dO
constexpr int kStageState = kStageOuts + kChunk * kOutBytes;
constexpr int kStageRows = kStageState + kWaves * 8 * kTileBytes;
constexpr int kStage = kStageRows + kWaves * 4 * kTileBytes;
static_assert(kHeadFactors <= 2 * kTileBytes, "the factors' tiles");
static_assert(kStage <= kLdsPerCu, "a compute unit's LDS");

// A workgroup takes 64 columns, two wavefronts for each 16: one the chain, the other
// the operands' loads, the two products that need no state, and the stores.  5.5 us a
// chunk of 128 heads at once, bound by the 112 KiB a chunk and head that it stores (6.9
// with one wavefront for all of it), 4.7 of 32 heads.
__global__ __launch_bounds__(128 * kWaves) void delta_back_wide_kernel(BackArgs args) {
  __shared__ __align__(16) char stage[kStage];
  const RuleArgs& a = args.rule;
  const ChunkSpace& space = a.space;
  const int place = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = place % kWaves;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const uint32_t turn = blockIdx.x >> 3;  // slices of a head on one XCD, as forward
  Work w;
  if (!find_work(a, static_cast<uint64_t>(turn / kSlices) * 8 + (blockIdx.x & 7), w)) return;
  const uint32_t head = w.head, key_head = w.head / a.group;
  const uint32_t first_row = w.first_row, begin = w.begin, length = w.length;
  const uint32_t chunks = w.chunks;
  const int slice = kWaves * (turn % kSlices) + wave;
  f32x4* const state_cells =
      reinterpret_cast<f32x4*>(stage + kStageState) + wave * 8 * 64 + lane;
  f32x4* const row_cells = reinterpret_cast<f32x4*>(stage + kStageRows) + wave * 4 * 64 + lane;
  const int own = 4 * g + (r & 3);  // a lane's token of each tile, where it has one

  if (place >= kWaves) {
    const uint32_t stage_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) char*)&stage[0]));
    const uint32_t key_step = static_cast<uint32_t>(a.key_stride) * 2;
    const uint32_t out_step = space.value_heads * kDim * 2;
    const uint32_t linear = 16 * lane;
    const auto fetch_first = [&](uint32_t c) {
      const uint64_t token = begin + c * kChunk;
      const uint32_t last = min(length - c * kChunk, static_cast<uint32_t>(kChunk)) - 1;
      const char* k = reinterpret_cast<const char*>(a.keys + token * a.key_stride +
                                                    key_head * kDim);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        stage_rows(k, key_step, last, kWaves * i + wave, lane, stage_at + kStageKeys);
      }
      const char* block = space.value_block(first_row + c, head);
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const int at = kWaves * i + wave;
        const char* from = at < 2 ? block + at * kTileBytes
                                  : block + kSolveBack + (at - 2) * kTileBytes;
        stage_tile(from, linear, stage_at + at * kTileBytes);
      }
      const char* columns = space.key_block(first_row + c, key_head) + kQueryColumns;
#pragma unroll
      for (int i = 0; i < kKeyTiles / kWaves; ++i) {
        const int at = kWaves * i + wave;
        stage_tile(columns + at * kTileBytes, linear,
                   stage_at + kStageQueryColumns + at * kTileBytes);
      }
    };
    const auto fetch_columns = [&](uint32_t c) {
      const char* columns = space.key_block(first_row + c, key_head) + kKeyColumns;
#pragma unroll
      for (int i = 0; i < kKeyTiles / kWaves; ++i) {
        const int at = kWaves * i + wave;
        stage_tile(columns + at * kTileBytes, linear, stage_at + kStageColumns + at * kTileBytes);
      }
    };
    const auto fetch_read = [&](uint32_t c) {
      const char* block = space.value_block(first_row + c, head) + kReadBack;
#pragma unroll
      for (int i = 0; i < (3 * kTriangle + kWaves - 1) / kWaves; ++i) {  // the last one twice
        const int at = min(kWaves * i + wave, 3 * kTriangle - 1);
        stage_tile(block + at * kTileBytes, linear, stage_at + kStageRead + at * kTileBytes);
      }
      const uint32_t last = min(length - c * kChunk, static_cast<uint32_t>(kChunk)) - 1;
      const char* d = reinterpret_cast<const char*>(args.d_outputs) +
                      (begin + static_cast<uint64_t>(c) * kChunk) * out_step +
                      2 * (head * kDim) + kOutBytes * (turn % kSlices);
      constexpr int kLanes = kOutBytes / 16, kRows = 64 / kLanes;  // of one tile
#pragma unroll
      for (int i = 0; i < kChunk / kRows / kWaves; ++i) {
        const int at = kWaves * i + wave;
        const uint32_t row = min(static_cast<uint32_t>(kRows * at + lane / kLanes), last);
        stage_tile(d, row * out_step + 16 * (lane % kLanes),
                   stage_at + kStageOuts + at * kTileBytes);
      }
    };
    const uint4* const q_columns =
        reinterpret_cast<const uint4*>(stage + kStageQueryColumns) + lane;
    const uint4* const read_back = reinterpret_cast<const uint4*>(stage + kStageRead) + lane;
    const char* const outs = stage + kStageOuts + own * kOutBytes + 32 * wave + 2 * (r & 12);

    // dO of a chunk as an operand over its tokens (rows past its end are zeros), and
    // P^T dO, which the chain takes.
    uint4 d_part[2];
    const auto take_outputs = [&](uint32_t c) {
      const int tokens = min(static_cast<int>(length - c * kChunk), kChunk);
      uint2 x[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint2 run = *reinterpret_cast<const uint2*>(outs + 16 * t * kOutBytes);
        const bool live = 16 * t + own < tokens;
        x[t] = transpose_quad(make_uint2(live ? run.x : 0, live ? run.y : 0), lane);
      }
      d_part[0] = make_uint4(x[0].x, x[0].y, x[1].x, x[1].y);
      d_part[1] = make_uint4(x[2].x, x[2].y, x[3].x, x[3].y);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int step = upper_first(t); step < 2; ++step) {
          const int at = upper_tile(t, step);
          const uint4 parts[3] = {read_back[at * 64], read_back[(kTriangle + at) * 64],
                                  read_back[(2 * kTriangle + at) * 64]};
          v = mfma3(parts, d_part[step], v);
        }
        row_cells[64 * t] = v;
      }
    };
    if (chunks != 0) {
      fetch_read(chunks - 1);
      fetch_first(chunks - 1);
      stage_ready();
      take_outputs(chunks - 1);
    }
    for (uint32_t c = chunks; c-- > 0;) {
      // The first half is there, the second has been read.  Stores issued after the
      // tiles stay in flight (the last chunk's rows may be fewer).
      if (c + 2 < chunks) {
        stage_ready<8>();
      } else {
        stage_ready();
      }
      fetch_columns(c);
      if (c != 0) fetch_read(c - 1);
      float queries[4], strengths[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float* const factors = reinterpret_cast<const float*>(stage);
        queries[t] = factors[kReadQuery + 16 * t + own];
        strengths[t] = factors[4 * (16 * t + own) + kStrength];
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) {  // dS1
        store_run(space.state_gradient(first_row + c, head) + slice * slice_cells(8),
                  t * kTileBytes + linear, transpose_quad(state_cells[64 * t], lane));
      }
      {  // (exp(G) Q)^T dO
        f32x4 sum[8] = {};
#pragma unroll
        for (int step = 0; step < 2; ++step) {
          uint4 part[3];
          f32x4 p[2];
          float d[8];
          widen8(d_part[step], d);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const f32x4 q = of_rows(queries[2 * step + u]);
#pragma unroll
            for (int i = 0; i < 4; ++i) p[u][i] = q[i] * d[4 * u + i];
          }
          split3(p[0], p[1], part);
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            sum[t] = mfma3(q_columns[(2 * t + step) * 64], part, sum[t]);
          }
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) state_cells[64 * t] = sum[t];
      }
      // The second half, X and the sum are there, the first half has been read.
      stage_ready<8>();
      if (c != 0) fetch_first(c - 1);
      const int tokens = min(static_cast<int>(length - c * kChunk), kChunk);
      char* const d = reinterpret_cast<char*>(args.d_values) +
                      (begin + static_cast<uint64_t>(c) * kChunk) * out_step +
                      2 * (head * kDim + 16 * slice);
#pragma unroll
      for (int t = 0; t < 4; ++t) {  // X, and Y = b X
        const f32x4 x = row_cells[64 * t], b = of_rows(strengths[t]);
        store_run(space.error_gradient(first_row + c, head) + slice * slice_cells(4),
                  t * kTileBytes + linear, transpose_quad(x, lane));
        const uint2 run = transpose_quad(
            make_uint2(bf16_pair(b[0] * x[0], b[1] * x[1]), bf16_pair(b[2] * x[2], b[3] * x[3])),
            lane);
        if (16 * t + own < tokens) store_run(d, (16 * t + own) * out_step + 2 * (r & 12), run);
      }
      if (c != 0) take_outputs(c - 1);
    }
    return;
  }

  // The chain.
  f32x4 state[8];  // the state's gradient, rows as in the forward scan
  load_final(args.d_final, w.tile, 0, 16 * slice + r, g, state);
  const uint4* k_rows[4];
  row_operands(stage + kStageKeys, lane, k_rows);
  const uint4* const k_columns = reinterpret_cast<const uint4*>(stage + kStageColumns) + lane;
  const uint4* const solve = reinterpret_cast<const uint4*>(stage + kStageSolve) + lane;
  if (chunks != 0) exchange();  // the first chunk's operands
  for (uint32_t c = chunks; c-- > 0;) {
    uint4 part[4][3];
#pragma unroll
    for (int t = 0; t < 8; ++t) state_cells[64 * t] = state[t];
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      split3(state[2 * step], state[2 * step + 1], part[step]);
    }
    exchange();
    f32x4 factors[4];
    float carries[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      factors[t] = reinterpret_cast<const f32x4*>(stage)[16 * t + own];
      carries[t] = reinterpret_cast<const float*>(stage)[kCarry + 16 * t + own];
    }
    // V' = P^T dO + exp(G_63 - G) K dS1
    f32x4 v[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 read = row_cells[64 * t];
      f32x4 seen[2] = {};
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        const uint4 k = k_rows[step][256 * t];
#pragma unroll
        for (int p = 2; p >= 0; --p) seen[p & 1] = mfma(k, part[step][p], seen[p & 1]);
      }
      const f32x4 carry = of_rows(carries[t]);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[t][i] = fmaf(carry[i], seen[0][i] + seen[1][i], read[i]);
    }
    // X = V' + (N^T b) V'
    {
      uint4 part[2][3];
#pragma unroll
      for (int step = 0; step < 2; ++step) split3(v[2 * step], v[2 * step + 1], part[step]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int step = upper_first(t); step < 2; ++step) {
          uint4 n[3];
#pragma unroll
          for (int p = 0; p < 3; ++p) n[p] = solve[(p * kTriangle + upper_tile(t, step)) * 64];
          v[t] = mfma6(n, part[step], v[t]);
        }
        row_cells[64 * t] = v[t];
      }
    }
    exchange();
    // dS0
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const f32x4 sum = state_cells[64 * t];
#pragma unroll
      for (int i = 0; i < 4; ++i) state[t][i] = fmaf(factors[0][kWhole], state[t][i], sum[i]);
    }
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      uint4 by_key[3];
      f32x4 m[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = 2 * step + u;
        const f32x4 k = of_rows(factors[t][kStrength] * -factors[t][kReadKey]);
#pragma unroll
        for (int i = 0; i < 4; ++i) m[u][i] = k[i] * v[t][i];
      }
      split3(m[0], m[1], by_key);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        state[t] = mfma3(k_columns[(2 * t + step) * 64], by_key, state[t]);
      }
    }
  }

  store_initial(args.d_initial, w.tile, 0, 16 * slice + r, g, state);
}

// ------------------------------------------------------------ 16 columns

// A workgroup takes 16 columns.  Four wavefronts share the chain's products by token
// rows (or state rows), four the two products beside it in the same way and the stores,
// with three exchanges a chunk, as the forward scan's narrow form.  3.4 us a chunk.
__global__ __launch_bounds__(512) void delta_back_narrow_kernel(BackArgs args) {
  constexpr int kNarrow = kDim / 16;
  // Parts of dS1 (4 steps over the keys), of V' and of -exp(G) Y / |k| (2 steps over
  // the tokens), and the fp32 accumulators that pass between the two kinds of wavefront.
  __shared__ uint4 state_parts[4][3][64];
  __shared__ uint4 row_parts[2][3][64];
  __shared__ uint4 written_parts[2][3][64];
  __shared__ f32x4 state_cells[8][64], read_cells[8][64];  // dS1, (exp(G) Q)^T dO
  __shared__ f32x4 value_cells[4][64], error_cells[4][64];  // P^T dO, X
  const RuleArgs& a = args.rule;
  const ChunkSpace& space = a.space;
  const uint32_t turn = blockIdx.x >> 3;  // slices of a head on one XCD, as forward
  Work w;
  if (!find_work(a, static_cast<uint64_t>(turn / kNarrow) * 8 + (blockIdx.x & 7), w)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int rows = wave & 3;  // this wavefront's token rows, 16 rows..
  const int from = upper_first(rows);
  const int slice = turn % kNarrow, first_value = 16 * slice;
  const uint32_t key_head = w.head / a.group;
  const uint32_t length = w.length, chunks = w.chunks;
  const int own = 4 * g + (r & 3);
  const uint32_t mine = 16 * rows + own;  // the token whose factors it loads

  // Past the first chunk, the same again.
  uint64_t token = w.begin;
  uint32_t row = w.first_row, last = 0;
  const auto go_to = [&](uint32_t c) {
    token = w.begin + static_cast<uint64_t>(c) * kChunk;
    row = w.first_row + c;
    last = min(length - c * kChunk, static_cast<uint32_t>(kChunk)) - 1;
  };
  if (chunks != 0) go_to(chunks - 1);

  if (wave >= 4) {
    const uint32_t out_step = space.value_heads * kDim * 2;
    uint2 outs[4];          // dO: columns 4 (r / 4).. of tokens 16 t + own
    uint4 read_back[2][3];  // P^T
    uint4 q_columns[2][2];
    float queries[4], strength;
    uint32_t live;  // the last token of `outs`
    const auto fetch_outs = [&]() {
      const char* d = reinterpret_cast<const char*>(args.d_outputs) + token * out_step +
                      2 * (w.head * kDim + first_value);
      live = last;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        outs[t] = *reinterpret_cast<const uint2*>(
            d + (min(static_cast<uint32_t>(16 * t + own), last) * out_step + 2 * (r & 12)));
      }
      const uint4* p =
          reinterpret_cast<const uint4*>(space.value_block(row, w.head) + kReadBack);
#pragma unroll
      for (int step = 0; step < 2; ++step) {  // rows 32.. have no first step
        const int tile = upper_tile(rows, step < from ? from : step);
#pragma unroll
        for (int u = 0; u < 3; ++u) read_back[step][u] = p[(u * kTriangle + tile) * 64 + lane];
      }
    };
    const auto fetch_queries = [&]() {
      const uint4* q =
          reinterpret_cast<const uint4*>(space.key_block(row, key_head) + kQueryColumns);
      const float* factors = reinterpret_cast<const float*>(space.value_block(row, w.head));
#pragma unroll
      for (int step = 0; step < 2; ++step) {
#pragma unroll
        for (int u = 0; u < 2; ++u) q_columns[u][step] = q[(2 * (2 * rows + u) + step) * 64 + lane];
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) queries[t] = factors[kReadQuery + 16 * t + own];
      strength = factors[4 * mine + kStrength];
    };
    // dO as an operand over the tokens (rows past the end are zeros), and P^T dO.
    uint4 d_part[2];
    const auto take_outs = [&]() {
      uint2 x[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bool there = static_cast<uint32_t>(16 * t + own) <= live;
        x[t] = transpose_quad(make_uint2(there ? outs[t].x : 0, there ? outs[t].y : 0), lane);
      }
      d_part[0] = make_uint4(x[0].x, x[0].y, x[1].x, x[1].y);
      d_part[1] = make_uint4(x[2].x, x[2].y, x[3].x, x[3].y);
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (from == 0) v = mfma3(read_back[0], d_part[0], v);
      value_cells[rows][lane] = mfma3(read_back[1], d_part[1], v);
    };
    if (chunks != 0) {
      fetch_outs();
      fetch_queries();
      take_outs();
    }
    for (uint32_t c = chunks; c-- > 0;) {
      char* const d = reinterpret_cast<char*>(args.d_values) + token * out_step +
                      2 * (w.head * kDim + first_value);
      float* const end = space.state_gradient(row, w.head) + slice * slice_cells(8) +
                         2 * rows * 256 + 4 * lane;
      float* const x_rows =
          space.error_gradient(row, w.head) + slice * slice_cells(4) + rows * 256 + 4 * lane;
      const uint32_t here = last;
      if (c != 0) go_to(c - 1);
      exchange();
      // (exp(G) Q)^T dO of state tiles 2 rows and the next
      uint4 part[2][3];
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        f32x4 p[2];
        float x[8];
        widen8(d_part[step], x);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x4 q = of_rows(queries[2 * step + u]);
#pragma unroll
          for (int i = 0; i < 4; ++i) p[u][i] = q[i] * x[4 * u + i];
        }
        split3(p[0], p[1], part[step]);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int step = 0; step < 2; ++step) sum = mfma3(q_columns[u][step], part[step], sum);
        read_cells[2 * rows + u][lane] = sum;
      }
      const float b = strength;
      __builtin_amdgcn_sched_barrier(0);
      fetch_outs();
      fetch_queries();
      __builtin_amdgcn_sched_barrier(0);
      exchange();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        store_cells(end + 256 * u, transpose_quad(state_cells[2 * rows + u][lane], lane));
      }
      exchange();
      const f32x4 x = error_cells[rows][lane], by = of_rows(b);
      const uint2 run = transpose_quad(
          make_uint2(bf16_pair(by[0] * x[0], by[1] * x[1]), bf16_pair(by[2] * x[2], by[3] * x[3])),
          lane);
      store_cells(x_rows, transpose_quad(x, lane));
      if (mine <= here) *reinterpret_cast<uint2*>(d + (mine * out_step + 2 * (r & 12))) = run;
      if (c != 0) take_outs();
    }
    return;
  }

  // The chain: token rows 16 wave.., state tiles 2 wave and 2 wave + 1.
  f32x4 state[2];
  load_final(args.d_final, w.tile, 2 * wave, first_value + r, g, state);
  const uint32_t key_step = static_cast<uint32_t>(a.key_stride) * 2;
  uint4 k_rows[4], k_columns[2][2], solve[2][3];
  f32x4 factors;
  float carry;
  const auto fetch_keys = [&]() {
    const char* k = reinterpret_cast<const char*>(a.keys + token * a.key_stride +
                                                  key_head * kDim);
    const uint32_t at = min(static_cast<uint32_t>(16 * wave + r), last) * key_step + 16 * g;
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      k_rows[step] = *reinterpret_cast<const uint4*>(k + 64 * step + at);
    }
  };
  const auto fetch_solve = [&]() {
    const char* const block = space.value_block(row, w.head);
    const uint4* p = reinterpret_cast<const uint4*>(block + kSolveBack);
    factors = reinterpret_cast<const f32x4*>(block)[mine];
    carry = reinterpret_cast<const float*>(block)[kCarry + mine];
#pragma unroll
    for (int step = 0; step < 2; ++step) {  // rows 32.. have no first step
      const int tile = upper_tile(wave, step < from ? from : step);
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
  for (uint32_t c = chunks; c-- > 0;) {
    {  // dS1, and cut into parts
      uint4 part[3];
      split3(state[0], state[1], part);
#pragma unroll
      for (int p = 0; p < 3; ++p) state_parts[wave][p][lane] = part[p];
#pragma unroll
      for (int u = 0; u < 2; ++u) state_cells[2 * wave + u][lane] = state[u];
    }
    exchange();
    // V' = P^T dO + exp(G_63 - G) K dS1.  Loads and LDS reads in the forward scan's order.
    uint4 part_s[4][3];
#pragma unroll
    for (int p = 2; p >= 0; --p) {
#pragma unroll
      for (int step = 0; step < 4; ++step) part_s[step][p] = state_parts[step][p][lane];
    }
    f32x4 v = value_cells[wave][lane];
    __builtin_amdgcn_sched_barrier(0);
    fetch_columns();
    if (c != 0) go_to(c - 1);
    __builtin_amdgcn_sched_barrier(0);
    const f32x4 carried = of_rows(carry);
    const f32x4 written = of_rows(factors[kStrength] * -factors[kReadKey]);
    f32x4 seen[2] = {};
#pragma unroll
    for (int p = 2; p >= 0; --p) {
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        seen[step & 1] = mfma(k_rows[step], part_s[step][p], seen[step & 1]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fmaf(carried[i], seen[0][i] + seen[1][i], v[i]);
    uint2 half[3];
    split3_half(v, half);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      reinterpret_cast<uint2*>(&row_parts[wave >> 1][p][lane])[wave & 1] = half[p];
    }
    exchange();
    // X = V' + (N^T b) V'
    uint4 part_r[2][3];
#pragma unroll
    for (int p = 2; p >= 0; --p) {
#pragma unroll
      for (int step = 0; step < 2; ++step) part_r[step][p] = row_parts[step][p][lane];
    }
    __builtin_amdgcn_sched_barrier(0);
    fetch_keys();
    __builtin_amdgcn_sched_barrier(0);
    if (from == 0) {
      f32x4 more = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int y = 2; y >= 0; --y) {  // parts x and y with x + y <= 2
#pragma unroll
        for (int x = 2 - y; x >= 0; --x) {
          v = mfma(solve[0][x], part_r[0][y], v);
          more = mfma(solve[1][x], part_r[1][y], more);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += more[i];
    } else {
      v = mfma6(solve[1], part_r[1], v);
    }
    error_cells[wave][lane] = v;
    f32x4 scaled;
#pragma unroll
    for (int i = 0; i < 4; ++i) scaled[i] = written[i] * v[i];
    split3_half(scaled, half);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      reinterpret_cast<uint2*>(&written_parts[wave >> 1][p][lane])[wave & 1] = half[p];
    }
    const float whole = factors[kWhole];
    exchange();
    // dS0 = exp(G_63) dS1 + (exp(G) Q)^T dO - (exp(G) K)^T Y
    uint4 part_w[2][3];
#pragma unroll
    for (int p = 2; p >= 0; --p) {
#pragma unroll
      for (int step = 0; step < 2; ++step) part_w[step][p] = written_parts[step][p][lane];
    }
    const f32x4 read[2] = {read_cells[2 * wave][lane], read_cells[2 * wave + 1][lane]};
    __builtin_amdgcn_sched_barrier(0);
    fetch_solve();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) state[u][i] = fmaf(whole, state[u][i], read[u][i]);
    }
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
  }
  store_initial(args.d_initial, w.tile, 2 * wave, first_value + r, g, state);
}

// ------------------------------------------------------- q, k, g and b

constexpr int kThreads = 512;
constexpr int kWide = 68;  // fp32 a row of a 64 x 64 matrix
constexpr int kRowTiles = 16;  // operand tiles of 64 rows over the 128 values

// Eight neighbouring values of a row, as an operand's places of natural order.
__device__ __forceinline__ void split_row(const f32x4 (&x)[2], uint4 (&part)[3]) {
  split3(x[0], x[1], part);
}

__device__ __forceinline__ float sum16(float x) {  // over the 16 lanes of a DPP row
  x = add_partner<1>(x);
  x = add_partner<2>(x);
  x = add_partner<4>(x);
  return add_partner<8>(x);
}

// x of the lane `kCtrl`'s row shift names, 0 where that lies outside the 16 lanes.
template <int kCtrl>
__device__ __forceinline__ float shifted(float x) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(x), kCtrl, 0xF, 0xF, true));
}
constexpr int kDppUp = 0x110, kDppDown = 0x100;  // row_shr, row_shl: from lane - n, lane + n
__device__ __forceinline__ float sum_to_here(float x) {  // of lanes 0.. to this one
  x += shifted<kDppUp + 1>(x);
  x += shifted<kDppUp + 2>(x);
  x += shifted<kDppUp + 4>(x);
  return x + shifted<kDppUp + 8>(x);
}
__device__ __forceinline__ float sum_from_here(float x) {  // of this one to lane 15
  x += shifted<kDppDown + 1>(x);
  x += shifted<kDppDown + 2>(x);
  x += shifted<kDppDown + 4>(x);
  return x + shifted<kDppDown + 8>(x);
}

struct Gradient {
  // X and E cut into parts, 16 tiles a part; then the four kinds of F and H, 6 tiles
  // a part.
  union {
    uint4 rows[2][3][kRowTiles][64];
    uint4 kinds[4][3][kTriangle][64];
  };
  uint4 outs[kRowTiles][64];  // dO
  float f[kChunk][kWide];
  float h[kChunk][kWide];
  float factors[kFactors];
  float norms[3][kChunk];  // 1/|k|, scale/|q|, 1/|q|
  // Of the value head at work: exp(G), exp(G) b, exp(G_63 - G) b.
  float decays[3][kChunk];
  float along[4][kChunk];  // X.E by step
  float sums[2][8][kChunk];
  float ends[8];
  // What pairs of tokens add to dg, block by block: by column (its tokens after the pair's
  // first), by row, and the whole block's.
  float pairs_to[kBlocks][16], pairs_from[kBlocks][16], pairs[kBlocks];
};
static_assert(sizeof(Gradient) <= kLdsPerCu, "one workgroup a compute unit");

// One workgroup per chunk row and key head.  Wavefront w takes the keys of state tile w
// and all tokens, so that a state is loaded and cut into parts once.  X and E are cut
// once, by the wavefront that loads them, and so are F and H.
//
// 32 heads of 85 chunks take 260 us: 535 MB of S0, dS1, E and X (2.1 TB/s), 2,850 matrix
// instructions a chunk and head (a fifth of their rate).  The parts of X and E leave room
// for one workgroup a compute unit, whose phases (loads, F and H, the states' products,
// the kinds) wait for each other: loads take a third of a head's time and LDS reads as
// much.  The pairs' sums for dg take 18 us of it.  Measured without them (255 us then) and
// left out: the next head's X and E asked for a phase ahead in a loop over chunks (286 us, with
// the registers it takes), F and H dealt out evenly (274), two tiles of keys by two of
// tokens a wavefront (262, every state loaded and cut twice).
__global__ __launch_bounds__(kThreads) void delta_gradient_kernel(BackArgs args) {
  __shared__ __align__(16) Gradient s;
  const RuleArgs& a = args.rule;
  const ChunkSpace& space = a.space;
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, g = lane >> 4;
  const int first_wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t row = blockIdx.x / space.key_heads;
  const uint32_t head = blockIdx.x % space.key_heads;
  const uint64_t token_step = static_cast<uint64_t>(space.value_heads) * kDim;
  {  // tokens of no request: zeros, a share of them for each chunk row
    const uint32_t from = min(static_cast<uint32_t>(a.offsets[a.requests]), a.tokens);
    for (uint64_t token = from + static_cast<uint64_t>(row); token < a.tokens;
         token += space.rows) {
      for (uint32_t i = t; i < a.group * kDim; i += kThreads) {
        args.d_values[token * token_step + head * a.group * kDim + i] = 0;
      }
      if (t < kDim) {
        args.d_queries[(token * space.key_heads + head) * kDim + t] = 0;
        args.d_keys[(token * space.key_heads + head) * kDim + t] = 0;
      }
      for (uint32_t i = t; i < a.group; i += kThreads) {
        args.d_log_decay[token * space.value_heads + head * a.group + i] = 0.0f;
        args.d_beta[token * space.value_heads + head * a.group + i] = 0;
      }
    }
  }
  const int4 chunk = a.chunks[row];
  const int count = chunk_tokens(a, chunk);
  if (count == 0) return;
  const uint64_t first = chunk.y;
  const char* const keys = space.key_block(row, head);
  const uint32_t outs_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) char*)&s.outs[0][0]));
  if (t < 3 * kChunk) {
    s.norms[t / kChunk][t % kChunk] = reinterpret_cast<const float*>(keys + kNorms)[t];
  }

  const auto eight = [&](int which, int token) {  // a sum over the wavefronts
    return ((s.sums[which][0][token] + s.sums[which][1][token]) +
            (s.sums[which][2][token] + s.sums[which][3][token])) +
           ((s.sums[which][4][token] + s.sums[which][5][token]) +
            (s.sums[which][6][token] + s.sums[which][7][token]));
  };
  f32x4 d_q[4] = {}, d_k[4] = {};  // of the token tiles
  for (uint32_t member = 0; member < a.group; ++member) {
    const uint32_t value_head = head * a.group + member;
    // Taken afresh for each head: the addresses that follow from them would otherwise
    // be kept over the loop, in more registers than there are.
    int lane = t & 63, wave = first_wave;
    asm volatile("" : "+v"(lane), "+s"(wave));
    const int r = lane & 15, g = lane >> 4;
    const float* const s0 = space.state(row, value_head);
    const float* const s1 = space.state_gradient(row, value_head);
    const float* const errors = space.errors(row, value_head);
    const float* const xs = space.error_gradient(row, value_head);
    // X and E of units (token tile, step) `wave` and `wave` + 8.
    f32x4 x[2][2], e[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int unit = wave + 8 * u;
      const int at = cells_at(4, unit >> 2, r, g) + 2 * (unit & 3) * slice_cells(4);
      x[u][0] = load4(xs + at), x[u][1] = load4(xs + at + 16);
      e[u][0] = load4(errors + at), e[u][1] = load4(errors + at + 16);
    }
    f32x4 start[4][2], end_gradient[4][2];  // S0's and dS1's rows of the keys
    const auto load_rows = [&](const float* state, f32x4 (&cells)[4][2]) {
      const float* p = state + cells_at(8, wave, r, g);
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        cells[step][0] = load4(p + 2 * step * slice_cells(8));
        cells[step][1] = load4(p + 2 * step * slice_cells(8) + 16);
      }
    };
    if (member != 0) __syncthreads();  // the last head's values have been read
    {  // dO as an operand over the values: rows past the end repeat the last, and
       // meet rows of K and Q that are zeros
      const char* d = reinterpret_cast<const char*>(args.d_outputs + first * token_step +
                                                    value_head * kDim);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int unit = wave + 8 * u;
        const uint32_t token = min(16 * (unit >> 2) + r, count - 1);
        stage_tile(d + 64 * (unit & 3), token * static_cast<uint32_t>(token_step) * 2 + 16 * g,
                   outs_at + unit * kTileBytes);
      }
    }
    static_assert(kFactors == kThreads, "one a thread");
    s.factors[64 * wave + lane] = reinterpret_cast<const float*>(
        space.value_block(row, value_head))[64 * wave + lane];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int unit = wave + 8 * u;
      uint4 part[3];
      float along = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        along = fmaf(x[u][0][i], e[u][0][i], fmaf(x[u][1][i], e[u][1][i], along));
      }
      along = add_partner<32>(add_partner<16>(along));
      if (g == 0) s.along[unit & 3][16 * (unit >> 2) + r] = along;
      split_row(x[u], part);
#pragma unroll
      for (int p = 0; p < 3; ++p) s.rows[0][p][unit][lane] = part[p];
      split_row(e[u], part);
#pragma unroll
      for (int p = 0; p < 3; ++p) s.rows[1][p][unit][lane] = part[p];
    }
    stage_ready();
    // Products of unit rows for blocks `wave` and `wave` + 8, asked for ahead of S0: loads
    // come back in order.
    f32x4 qk[2], kk[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const f32x4* const dots = reinterpret_cast<const f32x4*>(
          keys + kDots + 2 * min(wave + 8 * u, kBlocks - 1) * kTileBytes);
      qk[u] = dots[lane], kk[u] = dots[64 + lane];
    }
    load_rows(s0, start);
    if (wave == 0) {
      const float b = s.factors[4 * lane + kStrength];
      const float decay = __builtin_amdgcn_exp2f(s.factors[kSum + lane]);
      s.decays[0][lane] = decay;
      s.decays[1][lane] = decay * b;
      s.decays[2][lane] = b * decay_between(s.factors[kSum + kChunk - 1],
                                         s.factors[kSumRest + kChunk - 1], s.factors[kSum + lane],
                                         s.factors[kSumRest + lane]);
    }

    // F and H, ten blocks (i, j), j <= i, of 16 x 16; the two beside them that an
    // operand tile holds are zeros.
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int block = wave + 8 * u;
      if (block >= 12) break;
      const int i = block < 1 ? 0 : block < 3 ? 1 : block < 6 ? 2 : block < 10 ? 3
                    : block == 10 ? 0 : 2;
      const int j = block < 10 ? block - i * (i + 1) / 2 : i + 1;
      f32x4 fx = {0.0f, 0.0f, 0.0f, 0.0f}, hx = fx;
      if (block < 10) {
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          const int at = 4 * i + step, to = 4 * j + step;
          uint4 x_part[3], e_part[3];
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            x_part[p] = s.rows[0][p][at][lane];
            e_part[p] = s.rows[1][p][to][lane];
          }
          fx = mfma3(s.outs[at][lane], e_part, fx);
          hx = mfma6(x_part, e_part, hx);
        }
      }
      const int column = 16 * j + r;
      const float b_column = s.factors[4 * column + kStrength];
      const float sum = s.factors[kSum + column], rest = s.factors[kSumRest + column];
      float to = 0.0f, whole = 0.0f;
      f32x4 from;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int line = 16 * i + 4 * g + c;
        const float decay =
            decay_between(s.factors[kSum + line], s.factors[kSumRest + line], sum, rest);
        const float f = column <= line ? decay * (fx[c] * b_column) : 0.0f;
        const float h =
            column < line ? decay * (s.factors[4 * line + kStrength] * hx[c] * b_column) : 0.0f;
        s.f[line][column] = f;
        s.h[line][column] = h;
        // The pairs of this row up to this column: they cross the tokens after it and,
        // within the row's block, up to the row.
        const float pair = column < line ? fmaf(f, qk[u][c], -(h * kk[u][c])) : 0.0f;
        const float upto = sum_to_here(pair);
        const float before = shifted<kDppUp + 1>(upto);
        to += column <= line ? before : 0.0f;
        from[c] = upto;  // in lane 15, the row's
        whole += upto;
      }
      to = add_partner<32>(add_partner<16>(to));
      whole = add_partner<32>(add_partner<16>(whole));
      if (block < kBlocks) {
        if (g == 0) s.pairs_to[block][r] = to;
        if (r == 15) {
          *reinterpret_cast<f32x4*>(&s.pairs_from[block][4 * g]) = from;
          if (g == 0) s.pairs[block] = whole;
        }
      }
    }

    // S0 dO and S0 X, then <dS1, S0> and dS1 E, of this wavefront's keys.
    load_rows(s1, end_gradient);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 read_q[4] = {}, read_k[4] = {}, written[4] = {};
    {
      uint4 part[4][3];
#pragma unroll
      for (int step = 0; step < 4; ++step) split_row(start[step], part[step]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          const int at = 4 * i + step;
          uint4 x_part[3];
#pragma unroll
          for (int p = 0; p < 3; ++p) x_part[p] = s.rows[0][p][at][lane];
          read_q[i] = mfma3(s.outs[at][lane], part[step], read_q[i]);
          read_k[i] = mfma6(x_part, part[step], read_k[i]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    float end = 0.0f;
#pragma unroll
    for (int step = 0; step < 4; ++step) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        end = fmaf(start[step][0][i], end_gradient[step][0][i], end);
        end = fmaf(start[step][1][i], end_gradient[step][1][i], end);
      }
    }
    end *= s.factors[kWhole];
    {
      uint4 part[4][3];
#pragma unroll
      for (int step = 0; step < 4; ++step) split_row(end_gradient[step], part[step]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          const int at = 4 * i + step;
          uint4 e_part[3];
#pragma unroll
          for (int p = 0; p < 3; ++p) e_part[p] = s.rows[1][p][at][lane];
          written[i] = mfma6(e_part, part[step], written[i]);
        }
      }
    }
    __syncthreads();  // f and h are whole, X's and E's parts have been read

    // The four kinds, six units each: F and H by rows (over the tokens before), their
    // transposes (over the tokens after), with the norms of what they meet.
#pragma unroll
    for (int u = 0; u < 3; ++u) {
      const int unit = wave + 8 * u, kind = unit / 6, at = unit % 6;
      const float(&m)[kChunk][kWide] = (kind & 1) ? s.h : s.f;
      f32x4 y[2];
      if (kind < 2) {
        const int tile = at < 2 ? at : 2 + ((at - 2) >> 1), step = at < 2 ? 0 : (at & 1);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int from = 32 * step + 16 * v + 4 * g;
          const f32x4 cells = load4(&m[16 * tile + r][from]), unit_k = load4(&s.norms[0][from]);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[v][i] = cells[i] * unit_k[i];
        }
      } else {
        const int tile = at < 4 ? at >> 1 : at - 2, step = at < 4 ? (at & 1) : 1;
        const float sign = kind == 3 ? -1.0f : 1.0f;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int from = 32 * step + 16 * v + 4 * g;
          const f32x4 unit_q = load4(&s.norms[kind == 3 ? 0 : 1][from]);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[v][i] = m[from + i][16 * tile + r] * (sign * unit_q[i]);
        }
      }
      uint4 part[3];
      split_row(y, part);
#pragma unroll
      for (int p = 0; p < 3; ++p) s.kinds[kind][p][at][lane] = part[p];
    }
    uint4 k_columns[2], q_columns[2];
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      const int at = (2 * wave + step) * kTileBytes + 16 * lane;
      k_columns[step] = *reinterpret_cast<const uint4*>(keys + kKeyColumns + at);
      q_columns[step] = *reinterpret_cast<const uint4*>(keys + kQueryColumns + at);
    }
    __syncthreads();

#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 by_query = {0.0f, 0.0f, 0.0f, 0.0f}, by_read = by_query, by_write = by_query;
      const auto add = [&](int kind, int at, const uint4& columns, f32x4& to) {
        const uint4 part[3] = {s.kinds[kind][0][at][lane], s.kinds[kind][1][at][lane],
                               s.kinds[kind][2][at][lane]};
        to = mfma3(part, columns, to);
      };
#pragma unroll
      for (int step = 0; step < lower_steps(i); ++step) {  // the tokens before
        add(0, lower_tile(i, step), k_columns[step], by_query);
        add(1, lower_tile(i, step), k_columns[step], by_read);
      }
#pragma unroll
      for (int step = upper_first(i); step < 2; ++step) {  // the tokens after
        add(2, upper_tile(i, step), q_columns[step], by_write);
        add(3, upper_tile(i, step), k_columns[step], by_write);
      }
      float cells_k[8], cells_q[8];
      widen8(k_columns[i >> 1], cells_k);
      widen8(q_columns[i >> 1], cells_q);
      const int from = 16 * i + 4 * g;
      const f32x4 k_unit = load4(&s.norms[0][from]), q_unit = load4(&s.norms[1][from]);
      const f32x4 decay = load4(&s.decays[0][from]), read_by = load4(&s.decays[1][from]);
      const f32x4 kept = load4(&s.decays[2][from]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float dq = fmaf(decay[j], read_q[i][j], by_query[j]);
        const float seen = read_by[j] * read_k[i][j];
        const float carried = kept[j] * written[i][j];
        const float k = k_unit[j] * cells_k[4 * (i & 1) + j];
        const float q = q_unit[j] * cells_q[4 * (i & 1) + j];
        d_q[i][j] += dq;
        d_k[i][j] += (carried + by_write[j]) - (seen + by_read[j]);
        const float first = sum16(fmaf(q, decay[j] * read_q[i][j], -(k * seen)));
        const float last = sum16(k * carried);
        if (r == 0) {
          s.sums[0][wave][from + j] = first;
          s.sums[1][wave][from + j] = last;
        }
      }
    }
    end = wave_sum_valu(end);
    if (lane == 0) s.ends[wave] = end;
    __syncthreads();
    if (wave == 0) {
      const int tile = lane >> 4, place = lane & 15;
      const auto of = [](float x, int from) {
        return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), from));
      };
      // What S0 gives to this token and those after it.
      float from_start = sum_from_here(eight(0, lane));
      {
        const float second = of(from_start, 16), third = of(from_start, 32), fourth = of(from_start, 48);
        from_start += tile == 0 ? (second + third) + fourth
                : tile == 1 ? third + fourth
                : tile == 2 ? fourth : 0.0f;
      }
      // What the tokens before it give to dS1.
      float to_end = sum_to_here(eight(1, lane));
      {
        const float first_three[3] = {of(to_end, 15), of(to_end, 31), of(to_end, 47)};
        const float before = tile == 0 ? 0.0f
                             : tile == 1 ? first_three[0]
                             : tile == 2 ? first_three[0] + first_three[1]
                             : (first_three[0] + first_three[1]) + first_three[2];
        to_end = shifted<kDppUp + 1>(to_end) + before;
      }
      // Between tokens: pairs whose first is in this token's tile of 16, whose second is,
      // and, for the two tiles in the middle, whose ends lie on either side of it.
      float between = 0.0f, from = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= tile) between += s.pairs_to[i * (i + 1) / 2 + tile][place];
        if (i < tile) from += s.pairs_from[tile * (tile + 1) / 2 + i][place];
      }
      between += sum_from_here(from);
      if (tile == 1) between += s.pairs[3] + s.pairs[6];
      if (tile == 2) between += s.pairs[6] + s.pairs[7];
      const float ends = ((s.ends[0] + s.ends[1]) + (s.ends[2] + s.ends[3])) +
                         ((s.ends[4] + s.ends[5]) + (s.ends[6] + s.ends[7]));
      const float total = (ends + between) + (from_start + to_end);
      const float b = (s.along[0][lane] + s.along[1][lane]) + (s.along[2][lane] + s.along[3][lane]);
      if (lane < count) {
        const uint64_t at = (first + lane) * space.value_heads + value_head;
        args.d_log_decay[at] = total;
        args.d_beta[at] = static_cast<bf16_bits>(bf16_pair(b, 0.0f));
      }
    }
  }

  const int wave = first_wave;
  // Through the norms: with u = scale / |q|, d(raw) = u dq - q (u q.dq) / |q|^2, and
  // for keys the same with scale 1.
  float cells_k[2][8], cells_q[2][8];
#pragma unroll
  for (int step = 0; step < 2; ++step) {
    const int at = (2 * wave + step) * kTileBytes + 16 * lane;
    widen8(*reinterpret_cast<const uint4*>(keys + kKeyColumns + at), cells_k[step]);
    widen8(*reinterpret_cast<const uint4*>(keys + kQueryColumns + at), cells_q[step]);
  }
  __syncthreads();  // the last head's sums have been read
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float q = sum16(cells_q[i >> 1][4 * (i & 1) + j] * d_q[i][j]);
      const float k = sum16(cells_k[i >> 1][4 * (i & 1) + j] * d_k[i][j]);
      if (r == 0) {
        s.sums[0][wave][16 * i + 4 * g + j] = q;
        s.sums[1][wave][16 * i + 4 * g + j] = k;
      }
    }
  }
  __syncthreads();
  // What of a token's gradients lies along its q and k, once for all wavefronts.
  if (t < kChunk) {
    const float k_unit = s.norms[0][t], q_unit = s.norms[1][t];
    s.along[0][t] = a.normalize ? eight(0, t) * q_unit * s.norms[2][t] * s.norms[2][t] : 0.0f;
    s.along[1][t] = a.normalize ? eight(1, t) * k_unit * k_unit * k_unit : 0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int from = 16 * i + 4 * g;
    const f32x4 k_unit = load4(&s.norms[0][from]), q_unit = load4(&s.norms[1][from]);
    const f32x4 q_along = load4(&s.along[0][from]), k_along = load4(&s.along[1][from]);
    f32x4 dq, dk;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      dq[j] = fmaf(-cells_q[i >> 1][4 * (i & 1) + j], q_along[j], q_unit[j] * d_q[i][j]);
      dk[j] = fmaf(-cells_k[i >> 1][4 * (i & 1) + j], k_along[j], k_unit[j] * d_k[i][j]);
    }
    // Four tokens by four keys of a quad, transposed: lane 4 m + j gets token j's keys
    // state_key(wave, 4 m)..
    const uint2 q_run =
        transpose_quad(make_uint2(bf16_pair(dq[0], dq[1]), bf16_pair(dq[2], dq[3])), lane);
    const uint2 k_run =
        transpose_quad(make_uint2(bf16_pair(dk[0], dk[1]), bf16_pair(dk[2], dk[3])), lane);
    const int token = from + (r & 3);
    if (token < count) {
      const uint64_t at = ((first + token) * space.key_heads + head) * kDim +
                          state_key(wave, r & 12);
      *reinterpret_cast<uint2*>(args.d_queries + at) = q_run;
      *reinterpret_cast<uint2*>(args.d_keys + at) = k_run;
    }
  }
}

}  // namespace
}  // namespace gdn

extern "C" int32_t statecentric_gdn_state_codec_gated_delta_backward_launch_v1(
    void* stream, const gdn_state_codec_rule* rule, const uint16_t* d_outputs,
    const float* d_final, uint16_t* d_queries, uint16_t* d_keys, uint16_t* d_values,
    float* d_log_decay, uint16_t* d_beta, float* d_initial) {
  gdn::BackArgs args{};
  if (!gdn::rule_args(rule, true, args.rule) ||
      !gdn::token_rows(rule->tokens, d_outputs, d_queries, d_keys, d_values, d_log_decay,
                       d_beta) ||
      !gdn::aligned16(d_outputs, d_final, d_queries, d_keys, d_values, d_log_decay, d_beta,
                      d_initial)) {
    return gdn::kStatusInvalidArgument;
  }
  args.d_outputs = d_outputs, args.d_final = d_final, args.d_initial = d_initial;
  args.d_queries = d_queries, args.d_keys = d_keys, args.d_values = d_values;
  args.d_log_decay = d_log_decay, args.d_beta = d_beta;
  const gdn::ChunkSpace& space = args.rule.space;
  const uint64_t items = static_cast<uint64_t>(rule->requests) * rule->value_heads;
  // The forward scan's rule: 32 heads of one request take 3.4 us a chunk in the narrow
  // form and 4.7 in the wide one.
  const bool narrow = items * (gdn::kDim / 16) <= gdn::kComputeUnits;
  const uint64_t scans = (items + 7) / 8 * 8 * (narrow ? gdn::kDim / 16 : gdn::kSlices);
  if (scans > gdn::kMaxGrid) return gdn::kStatusInvalidArgument;
  const int32_t status =
      gdn::launch(narrow ? gdn::delta_back_narrow_kernel : gdn::delta_back_wide_kernel,
                  dim3(static_cast<uint32_t>(scans)),
                  dim3(narrow ? 512 : 128 * gdn::kWaves), stream, args);
  return status != gdn::kStatusOk
             ? status
             : gdn::launch(gdn::delta_gradient_kernel, dim3(space.rows * space.key_heads),
                           dim3(gdn::kThreads), stream, args);
}
