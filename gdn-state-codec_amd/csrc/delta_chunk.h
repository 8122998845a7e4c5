// What the kernels of the gated delta rule's chunked form share: the arguments,
// the workspace, and fp32 products on the bf16 matrix cores.
//
// A chunk of 64 tokens with start state S0 (here [key][value]), log decays summed
// to G_i inside the chunk, unit keys k_i, scaled unit queries q_i, strengths b_i:
//   A_ij = exp(G_i - G_j) k_i.k_j (j < i),   P_ij = exp(G_i - G_j) q_i.k_j (j <= i)
//   R = V - exp(G) K S0,   (I + A b) E = R,   U = b E
//   O = exp(G) Q S0 + P U,   S1 = exp(G_63) S0 + sum_j exp(G_63 - G_j) k_j u_j^T.
// (I + A b)^-1 = I + N b with N strictly lower triangular and
//   N_i = -A_i - sum_(m<i) A_im b_m N_m,
// which needs no division by b.  N, P and the operands' layouts depend on no
// state, so one kernel forms them for all chunks at once (delta_prepare.hip);
// what is left runs chunk after chunk (delta_scan.hip), every column of the state
// by itself.
//
// Precision.  q, k, v and the outputs' gradients are bf16, exact as they are.
// fp32 values enter v_mfma_f32_16x16x32_bf16 as three bf16 parts that sum to
// them exactly (truncation: 8 significant bits each), so a product with a bf16
// operand takes 3 instructions and loses nothing, and a product of two fp32
// operands takes 6 (the parts left out are below 2^-24 of the product).
// Accumulators, states, sums and factors are fp32; the decays' running sums are
// fp64, so that exp(G_i - G_j) of neighbours keeps its accuracy where G is large.
//
// Layouts.  An operand tile is 64 lanes x 16 bytes: lane l holds row (or column)
// l & 15 and 8 places of the contraction.  Contractions over keys or tokens use
// places of one order: the 8 places of lane group g = l >> 4 of a 32-wide step s
// are 32 s + 4 g + {0..3} and 32 s + 16 + 4 g + {0..3}.  Those are exactly the
// rows that group g holds of two accumulator tiles (rows 4 g + r), so a product's
// accumulators, cut into parts, are the next product's operand with no exchange
// between lanes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "activations.h"
#include "bf16_operands.h"
#include "gdn_state_codec_layer.h"
#include "launch.h"

namespace gdn {

constexpr int kChunk = GDN_STATE_CODEC_CHUNK;
constexpr float kUnitEps = 1e-6f;  // inside the square root of q's and k's norms

// Operand tiles of one chunk and key head: K and Q (rows = tokens, contraction
// over keys; 4 row tiles x 4 steps), their transposes (rows = keys, contraction
// over tokens; 8 row tiles x 2 steps; Q's for training only).
constexpr int kTileBytes = 1024;
constexpr int kKeyTiles = 16;      // tiles of each of the four
// Triangular operands (rows = tokens, contraction over tokens): 6 of the 8 tiles
// hold anything.
constexpr int kTriangle = 6;
__device__ __forceinline__ constexpr int lower_tile(int row, int step) {
  return row < 2 ? row : 2 * row - 2 + step;  // (0,0) (1,0) (2,0) (2,1) (3,0) (3,1)
}
__device__ __forceinline__ constexpr int upper_tile(int row, int step) {
  return row < 2 ? 2 * row + step : row + 2;  // (0,0) (0,1) (1,0) (1,1) (2,1) (3,1)
}
__device__ __forceinline__ constexpr int lower_steps(int row) { return row < 2 ? 1 : 2; }
__device__ __forceinline__ constexpr int upper_first(int row) { return row < 2 ? 0 : 1; }

constexpr int kSolveParts = 3;  // parts of N (an fp32 operand)
constexpr int kReadParts = 2;   // parts of P b: the outputs it makes are bf16

// Factors of a chunk's tokens for one value head, fp32 [7][64].
enum : int {
  kReadKey = 0,    // exp(G_i) / |k_i|
  kReadQuery = 1,  // exp(G_i) scale / |q_i|
  kStrength = 2,   // b_i, 0 past the request's end
  kWrite = 3,      // exp(G_63 - G_j) / |k_j|
  kWhole = 4,      // exp(G_63), in every place
  kSum = 5,        // G_i, and below it what fp32 left of it
  kSumRest = 6,
  kFactors = 7
};

// Bytes of the workspace's parts.
constexpr uint64_t kHeadFactors = kFactors * kChunk * 4;
__host__ __device__ constexpr uint64_t key_block_bytes(bool train) {
  return train ? 4 * kKeyTiles * kTileBytes + 3 * kChunk * 4 : 3 * kKeyTiles * kTileBytes;
}
__host__ __device__ constexpr uint64_t value_block_bytes(bool train) {
  const uint64_t serving = (kSolveParts + kReadParts) * kTriangle * kTileBytes + kHeadFactors;
  return train ? serving + 2 * kSolveParts * kTriangle * kTileBytes : serving;
}

// One chunk's key block, value block and, for training, states and rows.
struct ChunkSpace {
  char* base;
  uint32_t rows, key_heads, value_heads;
  bool train;

  __host__ __device__ uint64_t values_at() const {
    return static_cast<uint64_t>(rows) * key_heads * key_block_bytes(train);
  }
  __host__ __device__ uint64_t states_at() const {
    return values_at() + static_cast<uint64_t>(rows) * value_heads * value_block_bytes(train);
  }
  // Training: the start state and the end state's gradient of each chunk and
  // value head (fp32 [key][value]), then E and X (fp32 [64][128] each).
  // (1 KiB more: a block is read in whole tiles.)
  __host__ __device__ uint64_t total() const {
    return states_at() + (train ? static_cast<uint64_t>(rows) * value_heads *
                                      (2 * kTile + 2 * kChunk * kDim) * 4
                                : 0) +
           kTileBytes;
  }
  __device__ char* key_block(uint32_t row, uint32_t head) const {
    return base + (static_cast<uint64_t>(row) * key_heads + head) * key_block_bytes(train);
  }
  __device__ char* value_block(uint32_t row, uint32_t head) const {
    return base + values_at() +
           (static_cast<uint64_t>(row) * value_heads + head) * value_block_bytes(train);
  }
  __device__ float* state(uint32_t row, uint32_t head) const {
    return reinterpret_cast<float*>(base + states_at()) +
           (static_cast<uint64_t>(row) * value_heads + head) * (2 * kTile + 2 * kChunk * kDim);
  }
  __device__ float* state_gradient(uint32_t row, uint32_t head) const {
    return state(row, head) + kTile;
  }
  __device__ float* errors(uint32_t row, uint32_t head) const {
    return state(row, head) + 2 * kTile;
  }
  __device__ float* error_gradient(uint32_t row, uint32_t head) const {
    return state(row, head) + 2 * kTile + kChunk * kDim;
  }
};
// Places inside a key block.
constexpr int kKeyRows = 0;
constexpr int kQueryRows = kKeyTiles * kTileBytes;
constexpr int kKeyColumns = 2 * kKeyTiles * kTileBytes;
constexpr int kQueryColumns = 3 * kKeyTiles * kTileBytes;  // training
constexpr int kNorms = 4 * kKeyTiles * kTileBytes;  // training: fp32 1/|k|, scale/|q|, 1/|q|
// Places inside a value block: factors, N, P b, then N^T and P^T (training).
constexpr int kSolve = kHeadFactors;
constexpr int kReadOut = kSolve + kSolveParts * kTriangle * kTileBytes;
constexpr int kSolveBack = kReadOut + kReadParts * kTriangle * kTileBytes;
constexpr int kReadBack = kSolveBack + kSolveParts * kTriangle * kTileBytes;

struct RuleArgs {
  const bf16_bits* queries;
  const bf16_bits* keys;
  const bf16_bits* values;
  const float* log_decay;
  const bf16_bits* beta;
  uint64_t query_stride, key_stride, value_stride;
  const int32_t* offsets;
  const int32_t* chunk_offsets;
  const int4* chunks;
  const int32_t* order;
  uint32_t requests, tokens, group;
  float scale;
  uint32_t normalize;
  ChunkSpace space;
};

// Tokens of chunk row `row`, none where the tables point outside the batch.
__device__ __forceinline__ int chunk_tokens(const RuleArgs& a, const int4& chunk) {
  if (chunk.x < 0 || chunk.y < 0 || static_cast<uint32_t>(chunk.y) >= a.tokens) return 0;
  return min(min(max(chunk.z, 0), kChunk), static_cast<int>(a.tokens - chunk.y));
}

__device__ __forceinline__ f32x4 mfma(const uint4& a, const uint4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float upper(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
}

// Three parts of a pair: each the upper half of what the ones before left over
// (8 significant bits at a time, so the third is exact and their sum is x).
__device__ __forceinline__ void split3_pair(float x, float y, uint32_t& a, uint32_t& b,
                                            uint32_t& c) {
  a = upper_halves(__float_as_uint(x), __float_as_uint(y));
  x -= upper(x), y -= upper(y);
  b = upper_halves(__float_as_uint(x), __float_as_uint(y));
  x -= upper(x), y -= upper(y);
  c = upper_halves(__float_as_uint(x), __float_as_uint(y));
}

// The parts of 8 places of a contraction: two accumulator tiles, or 8 values.
__device__ __forceinline__ void split3(const f32x4& x, const f32x4& y, uint4 (&part)[3]) {
  split3_pair(x[0], x[1], part[0].x, part[1].x, part[2].x);
  split3_pair(x[2], x[3], part[0].y, part[1].y, part[2].y);
  split3_pair(y[0], y[1], part[0].z, part[1].z, part[2].z);
  split3_pair(y[2], y[3], part[0].w, part[1].w, part[2].w);
}

// c + a b of two fp32 operands in parts.
__device__ __forceinline__ f32x4 mfma6(const uint4 (&a)[3], const uint4 (&b)[3], f32x4 c) {
  c = mfma(a[0], b[2], c);
  c = mfma(a[1], b[1], c);
  c = mfma(a[2], b[0], c);
  c = mfma(a[0], b[1], c);
  c = mfma(a[1], b[0], c);
  return mfma(a[0], b[0], c);
}
// c + a b of an exact operand and an fp32 one.
__device__ __forceinline__ f32x4 mfma3(const uint4& a, const uint4 (&b)[3], f32x4 c) {
  c = mfma(a, b[2], c);
  c = mfma(a, b[1], c);
  return mfma(a, b[0], c);
}
__device__ __forceinline__ f32x4 mfma3(const uint4 (&a)[3], const uint4& b, f32x4 c) {
  c = mfma(a[2], b, c);
  c = mfma(a[1], b, c);
  return mfma(a[0], b, c);
}

__device__ __forceinline__ f32x4 load4(const float* p) {
  return *reinterpret_cast<const f32x4*>(p);
}

// Four neighbouring cells of a state.
__device__ __forceinline__ f32x4 load_cells(const float* p) { return load4(p); }
__device__ __forceinline__ f32x4 load_cells(const bf16_bits* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  return f32x4{widen_low(w.x), widen_high(w.x), widen_low(w.y), widen_high(w.y)};
}
__device__ __forceinline__ void store_cells(float* p, const f32x4& x) {
  *reinterpret_cast<f32x4*>(p) = x;
}
__device__ __forceinline__ void store_cells(bf16_bits* p, const f32x4& x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]));
}

// One tile, 16 bytes a lane, from global memory into LDS at `to` (bytes, the same
// for the wavefront) without passing the registers.  The caller waits
// (stage_ready) before any lane reads it.
__device__ __forceinline__ void stage_tile(const char* tile, int lane, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(16 * lane), "s"(tile), "s"(to)
               : "memory");
}

// Every staged tile of the workgroup is in LDS, and the stage read before may be
// overwritten, after this.
__device__ __forceinline__ void stage_ready() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

}  // namespace gdn
