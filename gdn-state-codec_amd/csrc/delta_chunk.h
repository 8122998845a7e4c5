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
// them exactly (8 significant bits each), so a product with a bf16
// operand takes 3 instructions and loses nothing, and a product of two fp32
// operands takes 6 (the parts left out are below 2^-24 of the product).
// Accumulators, states, sums and factors are fp32; the decays' running sums are
// fp64, so that exp(G_i - G_j) of neighbours keeps its accuracy where G is large.
//
// Layouts.  An operand is 16 rows (or columns) by 32 places of a contraction: lane
// l holds row l & 15 and the 8 places of lane group g = l >> 4.  An accumulator
// tile gives lane l column l & 15 of rows 4 g .. 4 g + 3.  The places of group g in
// step s of a contraction are the rows it holds of accumulator tiles 2 s and
// 2 s + 1, so a product's accumulators, cut into parts, are the next product's
// operand as they are.  For tokens that makes them 32 s + 4 g + {0..3} and
// 32 s + 16 + 4 g + {0..3}; the rows of the state's tiles are keys in such an order
// (state_key) that they are keys 32 s + 8 g + {0..7}, 16 bytes of a row of q or k.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "activations.h"
#include "bf16_operands.h"
#include "gdn_state_codec_layer.h"
#include "lane_exchange.h"
#include "launch.h"

namespace gdn {

constexpr int kChunk = GDN_STATE_CODEC_CHUNK;
constexpr float kUnitEps = 1e-6f;  // inside the square root of q's and k's norms

// bf16 operand tiles (64 lanes x 16 bytes) of one chunk and key head: K^T (rows =
// keys in state order, contraction over tokens; 8 row tiles x 2 steps), and for
// training Q^T.
constexpr int kTileBytes = 1024;
constexpr int kKeyTiles = 16;
// Triangular operands (rows and contraction = tokens): 6 of the 8 tiles hold
// anything.  N b, N^T b and P^T are three bf16 parts, 18 KiB (cut once
// here instead of by every slice that reads them); P b is two, since the outputs it
// makes are bf16.
constexpr int kTriangle = 6;
constexpr int kTriangleBytes = 3 * kTriangle * kTileBytes;
constexpr int kReadOutBytes = 2 * kTriangle * kTileBytes;
__device__ __forceinline__ constexpr int lower_tile(int row, int step) {
  return row < 2 ? row : 2 * row - 2 + step;  // (0,0) (1,0) (2,0) (2,1) (3,0) (3,1)
}
__device__ __forceinline__ constexpr int upper_tile(int row, int step) {
  return row < 2 ? 2 * row + step : row + 2;  // (0,0) (0,1) (1,0) (1,1) (2,1) (3,1)
}
// Its blocks of 16 x 16 on and below the diagonal, (i, j) at i (i + 1) / 2 + j.
constexpr int kBlocks = 10;
__device__ __forceinline__ constexpr int lower_steps(int row) { return row < 2 ? 1 : 2; }
__device__ __forceinline__ constexpr int upper_first(int row) { return row < 2 ? 0 : 1; }

// Key of row `row` of the state's tile `tile`.
__device__ __forceinline__ constexpr int state_key(int tile, int row) {
  return 32 * (tile >> 1) + 8 * (row >> 2) + 4 * (tile & 1) + (row & 3);
}
// Token of place i of lane group g in step `step`.
__device__ __forceinline__ constexpr int token_place(int step, int g, int i) {
  return 32 * step + (i < 4 ? 4 * g + i : 12 + 4 * g + i);
}

// Factors of a chunk's tokens for one value head (fp32): four of each token side by
// side (the forward chain's), then four rows.
enum : int {
  kReadKey = 0,    // exp(G_i) / |k_i|
  kStrength = 1,   // b_i, 0 past the request's end
  kWrite = 2,      // exp(G_63 - G_j) b_j / |k_j|
  kWhole = 3,      // exp(G_63)
  kReadQuery = 4 * kChunk,           // exp(G_i) scale / |q_i|
  kSum = kReadQuery + kChunk,        // G_i / ln 2, and below it what fp32 left of it
  kSumRest = kSum + kChunk,
  kCarry = kSumRest + kChunk,        // exp(G_63 - G_j) / |k_j|
  kFactors = kCarry + kChunk
};

// Bytes of the workspace's parts.
constexpr int kHeadFactors = kFactors * 4;
__host__ __device__ constexpr uint64_t key_block_bytes(bool train) {
  return train ? 2 * kKeyTiles * kTileBytes + 3 * kChunk * 4 + 2 * kBlocks * kTileBytes
               : kKeyTiles * kTileBytes;
}
__host__ __device__ constexpr uint64_t value_block_bytes(bool train) {
  return kHeadFactors + kReadOutBytes + (train ? 3 : 1) * kTriangleBytes;
}
// Places inside a key block: K^T, then for training Q^T, the norms (fp32 1/|k|,
// scale/|q|, 1/|q|), and q_i.k_j and k_i.k_j of scaled unit rows (fp32 accumulators, the
// two of each block side by side).
constexpr int kKeyColumns = 0;
constexpr int kQueryColumns = kKeyTiles * kTileBytes;
constexpr int kNorms = 2 * kKeyTiles * kTileBytes;
constexpr int kDots = kNorms + 3 * kChunk * 4;
// Places inside a value block: factors, N b, P b, then for training N^T b and P^T.
constexpr int kSolve = kHeadFactors;
constexpr int kReadOut = kSolve + kTriangleBytes;
constexpr int kSolveBack = kReadOut + kReadOutBytes;
constexpr int kReadBack = kSolveBack + kTriangleBytes;

// A long sequence of few heads is served in segments (delta_scan.hip): states between
// them and their maps, at most as many as half the compute units of each.
constexpr uint32_t kSplitItems = 32;    // requests x heads at most
constexpr uint32_t kSplitChunks = 64;   // chunks of a request at least, on the average
constexpr uint32_t kMostSegments = 16;  // after the first
constexpr uint32_t kSegmentStates = kComputeUnits;

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
  // Training: the start state and the end state's gradient of each chunk and value
  // head (fp32, 8 tiles of keys), then E and X (4 tiles of tokens each), in cells_at's
  // order.
  // For serving, the states between segments, where there may be any.
  __host__ __device__ bool may_split() const {
    return !train && value_heads <= kSplitItems && rows >= kSplitChunks;
  }
  __host__ __device__ uint64_t total() const {
    return states_at() + (train ? static_cast<uint64_t>(rows) * value_heads *
                                      (2 * kTile + 2 * kChunk * kDim) * 4
                          : may_split() ? static_cast<uint64_t>(kSegmentStates) * kTile * 4
                                        : 0) +
           kTileBytes;  // blocks are read in whole tiles
  }
  __device__ float* segments() const { return reinterpret_cast<float*>(base + states_at()); }
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

// fp32 matrices that the scans leave to the gradients: 16 columns by 16 rows at a time,
// as a wavefront's accumulator tile gives them after transpose_quad, 16 bytes a lane:
// 1 KiB a store (rows of the whole matrix, 64 bytes of each a store, took 1.3 times as
// long).  The floats from one slice of 16 columns to the next, of `tiles` row tiles:
__host__ __device__ constexpr int slice_cells(int tiles) { return tiles * 256; }
// Columns 8 g .. 8 g + 3 of the first two slices in row r of a tile; columns 4 on are
// 16 floats on, columns 32 on two slices.
__device__ __forceinline__ int cells_at(int tiles, int tile, int r, int g) {
  return (g >> 1) * slice_cells(tiles) + tile * 256 + 64 * (r >> 2) + 32 * (g & 1) + 4 * (r & 3);
}

// The two inputs that are read element by element, which a slice of a batch may
// start anywhere.
inline bool element_aligned(const float* log_decay, const bf16_bits* beta) {
  return reinterpret_cast<uintptr_t>(log_decay) % sizeof(float) == 0 &&
         reinterpret_cast<uintptr_t>(beta) % sizeof(bf16_bits) == 0;
}

// Tensors of one row a token: all there, unless there are no tokens (an empty tensor has
// no address, and no kernel reads a row of it).
template <typename... Pointers>
inline bool token_rows(uint32_t tokens, const Pointers*... pointers) {
  return tokens == 0 || ((pointers != nullptr) && ...);
}

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

// Three parts of a pair, each what the ones before left over, rounded to bf16.  The
// rest x - part is v_dot2_f32_bf16 of the pair of parts with (-1, 0) or (0, -1), exact
// like the subtraction (the rest of a rounding fits fp32), so that a pair takes 7
// instructions; 8 significant bits a part leave nothing of fp32's 24 (checked over
// 2^22 values of every size: what three parts miss is where the third would be a
// denormal).  The two constants are kept in registers: as inline constants the
// instruction reads them as fp32.  A value above the largest bf16 (0x1.fep127), an
// infinity and a NaN make their pair's other value a NaN too, which the products they
// enter would do anyway.
__device__ __forceinline__ void split3_pair(float x, float y, uint32_t& a, uint32_t& b,
                                            uint32_t& c) {
  uint32_t first = 0x0000BF80u, second = 0xBF800000u;
  asm("" : "+s"(first), "+s"(second));
  const bf16x2_t minus_first = __builtin_bit_cast(bf16x2_t, first);
  const bf16x2_t minus_second = __builtin_bit_cast(bf16x2_t, second);
  bf16x2_t part = __builtin_convertvector((f32x2_t){x, y}, bf16x2_t);
  a = __builtin_bit_cast(uint32_t, part);
  x = __builtin_amdgcn_fdot2_f32_bf16(part, minus_first, x, false);
  y = __builtin_amdgcn_fdot2_f32_bf16(part, minus_second, y, false);
  part = __builtin_convertvector((f32x2_t){x, y}, bf16x2_t);
  b = __builtin_bit_cast(uint32_t, part);
  x = __builtin_amdgcn_fdot2_f32_bf16(part, minus_first, x, false);
  y = __builtin_amdgcn_fdot2_f32_bf16(part, minus_second, y, false);
  c = bf16_pair(x, y);
}

// The parts of 8 places of a contraction: two accumulator tiles, or 8 values.
__device__ __forceinline__ void split3(const f32x4& x, const f32x4& y, uint4 (&part)[3]) {
  split3_pair(x[0], x[1], part[0].x, part[1].x, part[2].x);
  split3_pair(x[2], x[3], part[0].y, part[1].y, part[2].y);
  split3_pair(y[0], y[1], part[0].z, part[1].z, part[2].z);
  split3_pair(y[2], y[3], part[0].w, part[1].w, part[2].w);
}

// The same of one accumulator tile: half of an operand's places.
__device__ __forceinline__ void split3_half(const f32x4& x, uint2 (&part)[3]) {
  split3_pair(x[0], x[1], part[0].x, part[1].x, part[2].x);
  split3_pair(x[2], x[3], part[0].y, part[1].y, part[2].y);
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

// A lane's four rows of an accumulator tile, from the quad of lanes that holds one
// each: lane 4 m + i has token i's factor.
template <int kCtrl>
__device__ __forceinline__ float quad(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), kCtrl, 0xF, 0xF, true));
}
__device__ __forceinline__ f32x4 of_rows(float x) {
  return f32x4{quad<0x00>(x), quad<0x55>(x), quad<0xAA>(x), quad<0xFF>(x)};
}

// A 4 x 4 block of bf16 over a quad of lanes, transposed: from lane j's column j
// (rows 0, 1 | 2, 3) to its row j (columns 0, 1 | 2, 3), and back.  It makes
// accumulator columns whole 8-byte runs of a row.
__device__ __forceinline__ uint2 transpose_quad(const uint2& x, int lane) {
  const uint32_t near = (lane & 1) ? 0x03020706u : 0x05040100u;
  const uint32_t px = __builtin_amdgcn_mov_dpp(x.x, kDppQuadSwap1, 0xF, 0xF, true);
  const uint32_t py = __builtin_amdgcn_mov_dpp(x.y, kDppQuadSwap1, 0xF, 0xF, true);
  const uint32_t u = __builtin_amdgcn_perm(px, x.x, near);
  const uint32_t v = __builtin_amdgcn_perm(py, x.y, near);
  const bool up = (lane & 2) != 0;
  const uint32_t got = __builtin_amdgcn_mov_dpp(up ? u : v, kDppQuadSwap2, 0xF, 0xF, true);
  return make_uint2(up ? got : u, up ? v : got);
}

// exp(G_i - G_j) from the sums in units of ln 2, on the transcendental unit (about
// an ulp).
__device__ __forceinline__ float decay_between(float sum_i, float rest_i, float sum_j,
                                               float rest_j) {
  return __builtin_amdgcn_exp2f((sum_i - sum_j) + (rest_i - rest_j));
}

// The same of fp32: from lane j's column j (rows 0..3) to its row j (columns 0..3).
__device__ __forceinline__ f32x4 transpose_quad(const f32x4& x, int lane) {
  const bool odd = (lane & 1) != 0, up = (lane & 2) != 0;
  const float a = quad<kDppQuadSwap1>(odd ? x[0] : x[1]);
  const float b = quad<kDppQuadSwap1>(odd ? x[2] : x[3]);
  // rows (0 or 1) and (2 or 3), two columns each
  const float u0 = odd ? a : x[0], u1 = odd ? x[1] : a;
  const float v0 = odd ? b : x[2], v1 = odd ? x[3] : b;
  const float c = quad<kDppQuadSwap2>(up ? u0 : v0);
  const float d = quad<kDppQuadSwap2>(up ? u1 : v1);
  return f32x4{up ? c : u0, up ? d : u1, up ? v0 : c, up ? v1 : d};
}

// One tile into LDS at `to` (bytes, the same for the wavefront), 16 bytes a lane at
// `from` plus its own byte offset, without passing the registers.  The caller waits
// (stage_ready) before any lane reads it.  M0 holds the LDS address; nothing else in
// the kernels that call this uses it.
__device__ __forceinline__ void stage_tile(const char* from, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(offset), "s"(from), "s"(to)
               : "memory");
}

// 64 rows of q or k (one head's 256 bytes each) in LDS: four whole rows a tile, `step`
// bytes apart at `from`, rows past `last` the last again.  A row's 16-byte pieces are
// exchanged by its place, p to p ^ (row & 15), so that 16 rows' pieces of one operand fall
// on different banks.  (A tile of 16 rows by 64 bytes takes the address unit twice as
// long.)
__device__ __forceinline__ void stage_rows(const char* from, uint32_t step, uint32_t last,
                                           int tile, int lane, uint32_t to) {
  const uint32_t row = 4 * tile + (lane >> 4);
  stage_tile(from, min(row, last) * step + 16 * ((lane & 15) ^ (row & 15)),
             to + tile * kTileBytes);
}
// A lane's places of row tile 0, step by step, of rows staged so; the next row tile is 256
// on.
__device__ __forceinline__ void row_operands(const char* rows, int lane,
                                             const uint4* (&operand)[4]) {
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int step = 0; step < 4; ++step) {
    operand[step] = reinterpret_cast<const uint4*>(rows) + 16 * r + ((4 * step + g) ^ r);
  }
}

// Every staged tile of the workgroup is in LDS, and the stage read before may be
// overwritten, after this.  `kAfter` memory operations that each wavefront has issued
// after its last tile (store_run's, so that their number is known) stay in flight.
template <int kAfter = 0>
__device__ __forceinline__ void stage_ready() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(kAfter) : "memory");
}

// One store of 16 or 8 bytes a lane, `offset` bytes from `to` (the same for the
// wavefront).  The s_nop keeps the next instruction off the registers it reads.  The
// wide one is nontemporal: training's states are read when the whole scan is done, and
// operands stay in the caches instead (a training pass of 5,298 tokens 647 us, else 662).
__device__ __forceinline__ void store_run(void* to, uint32_t offset, const f32x4& x) {
  asm volatile("global_store_dwordx4 %0, %1, %2 nt\n\ts_nop 1"
               :
               : "v"(offset), "v"(x), "s"(to)
               : "memory");
}
__device__ __forceinline__ void store_run(void* to, uint32_t offset, const uint2& x) {
  asm volatile("global_store_dwordx2 %0, %1, %2\n\ts_nop 1"
               :
               : "v"(offset), "v"(__builtin_bit_cast(uint64_t, x)), "s"(to)
               : "memory");
}

// LDS written before it may be read by the workgroup's other wavefronts after it.
// Loads and stores to global memory stay in flight.
__device__ __forceinline__ void exchange() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

}  // namespace gdn
