// The gated delta rule over a tree of drafted tokens of each request, read from its
// cached state, and that state after an accepted path.
//
// With S0 the cached state of one value head ([value][key]), G_t the sum of the log
// decays from it down to node t, b_t the write strength, unit keys k and scaled unit
// queries q, and i above t where i is on t's path:
//   r_t = b_t (v_t - exp(G_t) S0 k_t)
//   u_t = r_t - sum_(i above t) A_ti u_i,        A_ti = b_t exp(G_t - G_i) k_t . k_i
//   o_t = exp(G_t) S0 q_t + sum_(i above t, and t) M_ti u_i,  M_ti = exp(G_t - G_i) q_t . k_i
// and after the path down to node c
//   S = exp(G_c) S0 + sum_(i on the path) exp(G_c - G_i) u_i k_i^T.
// So the state is read once for all nodes, by S0 K^T and S0 Q^T; what the tree is enters
// by which cells of A and M are there.
//
// Products with the state are on the bf16 matrix cores: k and q are exact as they are
// (their norms are factors of the results), an fp32 state is three parts (delta_chunk.h),
// a bf16 one itself.  So are those of A's blocks below the diagonal and of M with u, and a
// commit's of u with k: A, M and u are fp32 in three parts each, and of the nine products
// of two such the six that fp32 has room for are summed, in fp32.  A's blocks on the
// diagonal alone are on the fp32 matrix cores, whose accumulators are the next product's
// operand as they are: their (I + A)^-1, 16 x 16, is formed by substitution, which is stable
// for any keys.
//
// Bad values.  A product takes every cell, also those that are zero, so a NaN or an
// infinity in A, M, r or u would reach every node.  Those cells are set to zero, and the
// nodes that they belong to noted, for their outputs and those below them.  u is looked at
// too: finite inputs may sum up to more than fp32 holds, and the parts of a value above the
// largest bf16 are no numbers.  Where the inverse of a block passes that range, which the
// writes themselves need not, the block is solved node by node.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "activations.h"
#include "delta_chunk.h"
#include "gdn_state_codec_layer.h"
#include "lane_exchange.h"
#include "launch.h"
#include "stream_memory.h"
#include "work_order.h"

namespace gdn {
namespace {

constexpr int kMaxNodes = GDN_STATE_CODEC_MAX_NODES;
// A workgroup takes one head of one request, a wavefront 16 rows of its state.  (With two
// wavefronts a workgroup, so four a head, one request's 32 heads are no faster: 6.8 us for a
// tree of 16 nodes either way, 8 requests' 13.9 against 8.1.)
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
static_assert(16 * kWaves == kDim, "a workgroup takes a whole head");
constexpr double kInverseLn2 = 1.4426950408889634074;
// exp of less is 0 in fp32; sums of it stay far from what fp64 cannot tell apart.
constexpr double kLeastLogDecay = -200.0;
constexpr float kLargest = 0x1.fffffep127f;
constexpr float kLargestPart = 0x1.fep127f;  // of what is cut into bf16 parts

struct DraftArgs {
  const bf16_bits* queries;
  const bf16_bits* keys;
  const bf16_bits* values;
  const float* log_decay;
  const bf16_bits* beta;
  uint64_t query_stride, key_stride, value_stride;
  const int32_t* parents;
  const int32_t* offsets;
  const int32_t* slot_ids;
  const int32_t* accepted;
  void* pool;
  bf16_bits* outputs;
  uint32_t tokens, slots, value_heads, group, max_nodes;
  float scale;
  uint32_t normalize;
};

// A lane's 8 keys of a row of the state, in steps of 32: an operand's places.
template <typename Pool>
struct Cells;

template <>
struct Cells<float> {
  static constexpr int kParts = 3;
  f32x4 x, y;
  __device__ __forceinline__ void load(const float* p) {
    x = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
    y = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + 4));
  }
  __device__ __forceinline__ void parts(uint4 (&part)[3]) const { split3(x, y, part); }
};

template <>
struct Cells<bf16_bits> {
  static constexpr int kParts = 1;
  uint4 w;
  __device__ __forceinline__ void load(const bf16_bits* p) {
    w = stream_load(reinterpret_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void parts(uint4 (&part)[1]) const { part[0] = w; }
};

__device__ __forceinline__ f32x4 product(const uint4& a, const uint4 (&b)[3], f32x4 c) {
  return mfma3(a, b, c);
}
__device__ __forceinline__ f32x4 product(const uint4& a, const uint4 (&b)[1], f32x4 c) {
  return mfma(a, b[0], c);
}

// c + a b of 16 places of a contraction.  c is no sum of mfma's: right behind an instruction
// of 32 places that leaves c in the same registers, this one misses the first two rows of four
// of its product (in 80% of 10^8 such pairs on all compute units), and the compiler puts no
// wait between the two.
typedef __attribute__((ext_vector_type(4))) short bf16x4_bits;
__device__ __forceinline__ f32x4 mfma_half(const uint2& a, const uint2& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(bf16x4_bits, a),
                                                   __builtin_bit_cast(bf16x4_bits, b), c, 0, 0,
                                                   0);
}

// A 16 x 16 block in LDS.  A row's four runs of four columns are rotated by its place, so
// that 16 rows' runs fall on different banks.
struct Block {
  float cells[256];
  __device__ __forceinline__ float& at(int row, int column) {
    return cells[16 * row + (column ^ (row & 12))];
  }
  __device__ __forceinline__ f32x4 run(int row, int column) const {
    return load4(&cells[16 * row + (column ^ (row & 12))]);
  }
};

// Whether all parts of x, and with them every product with 0, are numbers.
__device__ __forceinline__ bool in_range(float x) { return fabsf(x) <= kLargestPart; }
__device__ __forceinline__ float largest(float x, float y, float z) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(x, y), z);
}
__device__ __forceinline__ float largest(const f32x4& x) {  // NaN where a cell is
  return largest(largest(fabsf(x[0]), fabsf(x[1]), fabsf(x[2])), fabsf(x[3]), 0.0f);
}
__device__ __forceinline__ bool in_range(const f32x4& x) { return in_range(largest(x)); }

// N = (I + A)^-1 - I of a diagonal block, from -A^T (row m of `block`: column m of -A),
// column `column` by each lane that stores it:  N_i = -A_i - sum_(m<i) A_im N_m, one m
// after another, so that each step waits for one fma alone.  The other lanes compute
// whatever is there.  Returns whether the lane's column is in range.
__device__ __forceinline__ bool invert(const Block& block, Block& inverse, int column,
                                       bool stores) {
  f32x4 n[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) n[c] = block.run(column, 4 * c);
#pragma unroll
  for (int m = 0; m < 15; ++m) {
    const float done = n[m / 4][m % 4];
#pragma unroll
    for (int c = (m + 1) / 4; c < 4; ++c) {
      const f32x4 l = block.run(m, 4 * c);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (4 * c + u > m) n[c][u] = fmaf(l[u], done, n[c][u]);
      }
    }
  }
  // Formed here, not where it is stored: all rows would wait in registers.
#pragma unroll
  for (int c = 0; c < 4; ++c) asm volatile("" : "+v"(n[c]));
  wave_sync();  // `inverse` may be `block`
  if (stores) {
#pragma unroll
    for (int i = 0; i < 16; ++i) inverse.at(i, column) = n[i / 4][i % 4];
  }
  return in_range(f32x4{largest(n[0]), largest(n[1]), largest(n[2]), largest(n[3])});
}

// A value that all lanes share, known to be one.
__device__ __forceinline__ int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// The request's nodes: first token row and how many, 0 where there is nothing to do.
__device__ __forceinline__ int request_nodes(const DraftArgs& a, uint32_t r, int32_t& slot,
                                             uint64_t& begin) {
  slot = uniform(a.slot_ids[r]);
  const int32_t first = max(uniform(a.offsets[r]), 0);
  const int32_t last = static_cast<int32_t>(
      min(static_cast<int64_t>(uniform(a.offsets[r + 1])), static_cast<int64_t>(a.tokens)));
  begin = static_cast<uint32_t>(first);
  if (slot < 0 || static_cast<uint32_t>(slot) >= a.slots || last <= first) return 0;
  return min(last - first, static_cast<int32_t>(a.max_nodes));
}

// 16 bytes of a row of k or q (16 lanes a row), into LDS, and its sum of squares.  A row's
// pieces are exchanged by its place, p to p ^ (row & 15), so that 16 rows' pieces of one
// operand fall on different banks.
__device__ __forceinline__ float stage_piece(uint4* rows, int row, int piece, const uint4& w) {
  rows[16 * row + (piece ^ (row & 15))] = w;
  float x[8];
  widen8(w, x);
  return row_sum(dot8(x, x));
}
__device__ __forceinline__ const uint4& staged(const uint4* rows, int row, int piece) {
  return rows[16 * row + (piece ^ (row & 15))];
}

// Four tokens' values of a lane's column, from the four columns of one token of each
// lane of a quad.
__device__ __forceinline__ f32x4 value_columns(const uint2& w, int lane) {
  const uint2 t = transpose_quad(w, lane);
  return f32x4{widen_low(t.x), widen_high(t.x), widen_low(t.y), widen_high(t.y)};
}

// Sets the cells of a lane's column that are out of range to 0, and gives their nodes, a bit
// each, in all lanes of that column.
__device__ __forceinline__ uint32_t set_apart(f32x4& x, int lane) {
  uint32_t column = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (!in_range(x[c])) column |= 1u << (4 * (lane >> 4) + c), x[c] = 0.0f;
  }
  column |= __shfl_xor(column, 16);
  return column | __shfl_xor(column, 32);
}

// The same, after x <- (I + A)^-1 x of one block from -A^T, node after node: what an inverse
// past fp32's range cannot give.
__device__ __forceinline__ uint32_t solve_by_steps(const Block& block, f32x4& x, int lane) {
#pragma unroll 1
  for (int from = 0; from < 4; ++from) {  // the lane group that has the node
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float u = __shfl(x[c], 16 * from + (lane & 15));
      if (!in_range(u)) u = 0.0f;
      const f32x4 below = block.run(4 * from + c, 4 * (lane >> 4));
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = fmaf(below[i], u, x[i]);
    }
  }
  return set_apart(x, lane);
}

// u = x + N x of 16 nodes, and the nodes that are not in range (then 0), a bit each.  A cell
// of x or u that is out of range would reach every node through the zeros of the products
// it enters, so both are looked at, but u first: it is out of range wherever x or a cell of
// N is.
__device__ __forceinline__ uint32_t solve(const Block& inverse, const Block& block, int lane,
                                          f32x4& x) {
  const f32x4 n = inverse.run(lane & 15, 4 * (lane >> 4));
  const f32x4 u = block_product(n, x, x);
  uint32_t bad = 0;
  if (__any(!in_range(u))) {
    if (__any(!in_range(n))) {
      bad = solve_by_steps(block, x, lane);
    } else {
      bad = set_apart(x, lane);
      x = block_product(n, x, x);
      bad |= set_apart(x, lane);
    }
  } else {
    x = u;
  }
  return bad;
}

// -------------------------------------------------------------------- the tree

constexpr int blocks_of(int tiles) { return tiles * (tiles + 1) / 2; }
// Block (i, j <= i) of a lower triangular matrix.
__host__ __device__ constexpr int block_at(int i, int j) { return i * (i + 1) / 2 + j; }

// -A below the diagonal and M as operands of products with u, in three parts, row tile by
// row tile: blocks 2 s and 2 s + 1 of a row side by side (16 bytes a lane, the places of
// delta_chunk.h), a last one without a partner by itself (8 bytes a lane).  In units of 8
// bytes: a block takes 3 x 64, and block j of row tile i starts at
constexpr int kBlockPlaces = 3 * 64;
__host__ __device__ constexpr int step_at(int i, int j) {
  return (i * (i - 1) / 2 + j / 2 * 2) * kBlockPlaces;
}
__host__ __device__ constexpr int read_at(int i, int j) {
  return (i * (i + 1) / 2 + j / 2 * 2) * kBlockPlaces;
}
constexpr int step_places(int tiles) { return tiles > 1 ? step_at(tiles, 0) : 1; }
constexpr int read_places(int tiles) { return read_at(tiles, 0); }

// A block (an accumulator) as its part of such an operand, where it has a partner (then
// `second` is whether it is the second of the two) or not.
__device__ __forceinline__ void store_operand(uint2* operand, bool paired, bool second, int lane,
                                              const f32x4& block) {
  const f32x4 row = transpose_quad(block, lane);  // row 4 g + (r & 3), columns r & 12 ..
  uint2 part[3];
  split3_half(row, part);
  const int place = 4 * (lane >> 4) + (lane & 3) + 16 * (lane >> 2 & 3);
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    operand[paired ? 128 * p + 2 * place + (second ? 1 : 0) : 64 * p + place] = part[p];
  }
}

// Parts of u, tiles 2 s and 2 s + 1 side by side.
typedef uint4 Pair[3];

// c + (blocks 2 s, 2 s + 1 of a row) (u of those tiles).
__device__ __forceinline__ f32x4 add_pair(const uint2* operand, int lane, const Pair& u, f32x4 c) {
  uint4 a[3];
#pragma unroll
  for (int p = 0; p < 3; ++p) a[p] = reinterpret_cast<const uint4*>(operand)[64 * p + lane];
  return mfma6(a, u, c);
}
// c + (the last block of a row, that has no partner) (u of its tile), c no sum of add_pair's.
__device__ __forceinline__ f32x4 add_single(const uint2* operand, int lane, const Pair& u,
                                            f32x4 c) {
  uint2 a[3], b[3];
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    a[p] = operand[64 * p + lane];
    b[p] = make_uint2(u[p].x, u[p].y);
  }
  c = mfma_half(a[0], b[2], c);
  c = mfma_half(a[1], b[1], c);
  c = mfma_half(a[2], b[0], c);
  c = mfma_half(a[0], b[1], c);
  c = mfma_half(a[1], b[0], c);
  return mfma_half(a[0], b[0], c);
}

template <int kTiles>
struct TreeShared {
  static constexpr int kNodes = 16 * kTiles;
  union {
    struct {
      uint4 k[kNodes * 16], q[kNodes * 16];
    };
    uint4 out[kNodes * 16];       // once all products of k and q are formed
  };
  Block own[kTiles];              // on the diagonal: -A^T
  Block inverse[kTiles];          // and N
  alignas(16) uint2 step[step_places(kTiles)];  // -A below it
  alignas(16) uint2 read[read_places(kTiles)];  // M
  alignas(16) float k_square[kNodes], q_square[kNodes];
  // Factors of a node: of a key, -b / |k|, scale / |q|; then -b exp(G) / |k| of S0 k,
  // exp(G) scale / |q| of S0 q, and b.
  float k_unit[kNodes], k_step[kNodes], q_unit[kNodes];
  float seen[kNodes], look[kNodes], strength[kNodes];
  float sum[kNodes], rest[kNodes];       // G / ln 2, and what fp32 left of it
  uint64_t above[kNodes];
  uint32_t bad_node[2], bad_output[2];   // a bit a node
};

// What a node's path gives, one node a lane of one wavefront.  By doubling: after round i a
// lane's sum is of 2^i nodes up from its own.
struct Path {
  double sum;      // of log decays
  uint64_t above;  // a bit a node
  bool bad;        // the node's own log decay
};

__device__ __forceinline__ Path tree_path(int lane, int nodes, int parent, float log_decay) {
  const bool real = lane < nodes;
  int up = real && parent >= 0 && parent < lane ? parent : -1;
  Path p;
  p.above = up >= 0 ? 1ull << up : 0;
  p.bad = real && !(log_decay <= kLargest);
  p.sum = real && !p.bad ? fmax(static_cast<double>(log_decay), kLeastLogDecay) : 0.0;
  for (int reach = 1; reach < nodes; reach <<= 1) {
    const int from = up >= 0 ? up : lane;
    const double sum_up = __shfl(p.sum, from);
    const uint64_t above_up = __shfl(p.above, from);
    const int next = __shfl(up, from);
    if (up >= 0) {
      p.sum += sum_up;
      p.above |= above_up;
      up = next;
    }
  }
  p.sum *= kInverseLn2;
  return p;
}

template <int kTiles>
__device__ __forceinline__ void tree_tables(TreeShared<kTiles>& s, const DraftArgs& a, int lane,
                                            int nodes, const Path& p, float strength) {
  const uint64_t all_bad = __ballot(p.bad);
  if (lane < TreeShared<kTiles>::kNodes) {
    const float high = static_cast<float>(p.sum), low = static_cast<float>(p.sum - high);
    float k_unit = 1.0f, q_unit = a.scale;
    if (a.normalize) {
      k_unit = 1.0f / sqrtf(s.k_square[lane] + kUnitEps);
      q_unit *= 1.0f / sqrtf(s.q_square[lane] + kUnitEps);
    }
    const float decay = decay_between(high, low, 0.0f, 0.0f);
    const float b = lane < nodes ? strength : 0.0f;
    s.k_unit[lane] = k_unit;
    s.k_step[lane] = -b * k_unit;
    s.q_unit[lane] = q_unit;
    s.seen[lane] = -b * (decay * k_unit);
    s.look[lane] = decay * q_unit;
    s.strength[lane] = b;
    s.sum[lane] = high;
    s.rest[lane] = low;
    s.above[lane] = p.above;
  }
  if (lane < 2) {
    s.bad_node[lane] = static_cast<uint32_t>(all_bad >> (32 * lane));
    s.bad_output[lane] = 0;
  }
}

// 16 bytes of a token's row: `row` tokens after `base`, `step` elements apart.
__device__ __forceinline__ const void* row_at(const bf16_bits* base, uint32_t row, uint32_t step,
                                              uint32_t offset) {
  return reinterpret_cast<const char*>(base) + (row * step + offset) * 2u;
}

// The first wavefront forms the tables and inverts, the others form the nodes' products; the
// state's are between, wherever a wavefront would wait.
//
// What bounds it (32 heads): few nodes, latency around the bytes: 64 trees of 16 on an fp32
// pool take 32 us by the form of 16 nodes (three workgroups a compute unit), 35 by that of 64
// (two, so four rounds of the card), of which the bytes are 25.  Many nodes, a workgroup's
// phases, of which two share a compute unit: 256 trees of up to 48 nodes on a bf16 pool take
// 122 us (bytes 68), 128 chains of 64 on an fp32 pool 131 (bytes 77).  The matrix units are busy
// for 20 and 36% of that, wavefronts wait for 54 and 41% of their lives; the loads and stores
// without the rest take about 100 us, the rest without them as much.  A persistent workgroup
// that asks for the next head's nodes, 32 nodes at a time with less LDS, two heads a workgroup
// and launches of their own for the smaller trees of a batch are no faster.
//
// Four workgroups a compute unit for a bf16 pool's trees of up to 32 nodes: 64 registers, which
// the compiler is held to (it takes 66 otherwise: 256 trees 95 us, 91 so).
template <typename Pool, int kTiles>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(sizeof(Pool) == 2 && kTiles <= 2 ? 8 : 2)))
void tree_kernel(DraftArgs a) {
  constexpr int kNodes = 16 * kTiles;
  constexpr int kPasses = 2 * kNodes * 16 / kThreads;
  constexpr int kBlocks = blocks_of(kTiles);
  constexpr int kPairs = (kBlocks + kWaves - 2) / (kWaves - 1);
  __shared__ TreeShared<kTiles> s;

  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t head = static_cast<uint32_t>(xcd_contiguous_item(blockIdx.x, gridDim.x));
  const uint32_t n = head / a.value_heads, h = head % a.value_heads, hk = h / a.group;
  int32_t slot;
  uint64_t begin;
  const int nodes = request_nodes(a, n, slot, begin);
  if (nodes == 0) return;
  const int tiles = (nodes + 15) / 16;

  // Everything from memory is asked for here: the nodes first, which are waited for first.
  int parent = -1;
  float log_decay = 0.0f, strength = 0.0f;
  if (wave == 0 && lane < nodes) {
    const uint64_t first = begin * a.value_heads + h;
    parent = (a.parents + begin)[lane];
    log_decay = (a.log_decay + first)[lane * a.value_heads];
    strength = widen((a.beta + first)[lane * a.value_heads]);
  }
  const int piece = threadIdx.x & 15;
  const bf16_bits* const keys = a.keys + begin * a.key_stride + hk * kDim;
  const bf16_bits* const queries = a.queries + begin * a.query_stride + hk * kDim;
  const uint32_t key_step = static_cast<uint32_t>(a.key_stride);
  const uint32_t query_step = static_cast<uint32_t>(a.query_stride);
  uint4 pieces[kPasses];  // the keys', then the queries'
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    // The same for a wavefront, like the row's tile.
    const int place = p * (kThreads / 16) + 4 * wave;
    const bool query = place >= kNodes;
    const int first = place % kNodes;
    if (first < 16 * tiles) {
      const uint32_t row = min(first + g, nodes - 1);
      pieces[p] = *static_cast<const uint4*>(
          row_at(query ? queries : keys, row, query ? query_step : key_step, 8 * piece));
    }
  }
  const int first_row = 16 * wave;
  uint2 v[kTiles];
  {
    const bf16_bits* const values = a.values + begin * a.value_stride + h * kDim + first_row;
    const uint32_t step = static_cast<uint32_t>(a.value_stride);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      if (i < tiles) {
        const uint32_t row = min(16 * i + 4 * g + (r & 3), nodes - 1);
        v[i] = *static_cast<const uint2*>(row_at(values, row, step, r & 12));
      }
    }
  }
  Cells<Pool> cells[4];
  {
    const Pool* const state = static_cast<const Pool*>(a.pool) +
                              (static_cast<uint64_t>(slot) * a.value_heads + h) * kTile +
                              first_row * kDim;
    const uint32_t place = r * kDim + 8 * g;
#pragma unroll
    for (int step = 0; step < 4; ++step) cells[step].load(state + (place + 32 * step));
  }

  Path path;
  if (wave == 0) path = tree_path(lane, nodes, parent, log_decay);
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int place = p * (kThreads / 16) + 4 * wave;
    const bool query = place >= kNodes;
    const int first = place % kNodes;
    if (first < 16 * tiles) {
      const float square = stage_piece(query ? s.q : s.k, first + g, piece, pieces[p]);
      if (piece == 0) (query ? s.q_square : s.k_square)[first + g] = square;
    }
  }
  exchange();

  f32x4 seen[kTiles], read[kTiles];  // S0 K^T and S0 Q^T, a token a row
  auto state_products = [&]() {
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kTiles; ++i) seen[i] = read[i] = zero;
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      uint4 part[Cells<Pool>::kParts];
      cells[step].parts(part);
      const uint4* const k = &staged(s.k, r, 4 * step + g);
      const uint4* const q = &staged(s.q, r, 4 * step + g);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        if (i < tiles) {
          seen[i] = product(k[256 * i], part, seen[i]);
          read[i] = product(q[256 * i], part, read[i]);
        }
      }
    }
  };

  if (wave == 0) {
    tree_tables(s, a, lane, nodes, path, strength);
    exchange();
    state_products();
    exchange();
    const int diagonal = min(g, kTiles - 1);
    invert(s.own[diagonal], s.inverse[diagonal], r, g < tiles);
    exchange();
  } else {
    f32x4 kk[kPairs], qk[kPairs];
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      const int block = wave - 1 + e * (kWaves - 1);
      const int i = block < 1 ? 0 : block < 3 ? 1 : block < 6 ? 2 : 3;
      const int j = block - block_at(i, 0);
      kk[e] = qk[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (block < kBlocks && i < tiles) {
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          const uint4* const k = &staged(s.k, r, 4 * step + g);
          const uint4* const q = &staged(s.q, r, 4 * step + g);
          const uint4 column = k[256 * j];
          kk[e] = mfma(k[256 * i], column, kk[e]);
          qk[e] = mfma(q[256 * i], column, qk[e]);
        }
      }
    }
    exchange();
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      const int block = wave - 1 + e * (kWaves - 1);
      const int i = block < 1 ? 0 : block < 3 ? 1 : block < 6 ? 2 : 3;
      const int j = block - block_at(i, 0);
      if (block < kBlocks && i < tiles) {
        const int first = 16 * i + 4 * g, column = 16 * j + r;
        const float sum_c = s.sum[column], rest_c = s.rest[column], unit_c = s.k_unit[column];
        // The rows' factors: a row at a time where registers, not LDS, decide how many
        // workgroups share a compute unit (four then on a bf16 pool: 256 trees of 16 nodes
        // take 68.6 us, with all rows' at once 75); else at once (the trees of up to 48 nodes
        // 121 us, a row at a time 125).
        constexpr bool kAtOnce = kTiles > 2;
        f32x4 sum, rest, k_step, q_unit;
        if (kAtOnce) {
          sum = load4(&s.sum[first]), rest = load4(&s.rest[first]);
          k_step = load4(&s.k_step[first]), q_unit = load4(&s.q_unit[first]);
        }
        float worst = 0.0f;
        f32x4 x, y;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int row = first + c;
          const bool up = (s.above[row] >> column & 1) != 0;
          const bool self = row == column && column < nodes;
          if (!kAtOnce) {
            sum[c] = s.sum[row], rest[c] = s.rest[row];
            k_step[c] = s.k_step[row], q_unit[c] = s.q_unit[row];
          }
          const float decay = decay_between(sum[c], rest[c], sum_c, rest_c) * unit_c;
          x[c] = up ? decay * k_step[c] * kk[e][c] : 0.0f;
          y[c] = up || self ? decay * q_unit[c] * qk[e][c] : 0.0f;
          worst = largest(worst, fabsf(x[c]), fabsf(y[c]));
          if (!kAtOnce) __builtin_amdgcn_sched_barrier(0);
        }
        if (__any(!in_range(worst))) {
          uint32_t bad_node = 0, bad_output = 0;  // a bit a row
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (!in_range(x[c])) bad_node |= 1u << c, x[c] = 0.0f;
            if (!in_range(y[c])) bad_output |= 1u << c, y[c] = 0.0f;
          }
          if (bad_node) atomicOr(&s.bad_node[first >> 5], bad_node << (first & 31));
          if (bad_output) atomicOr(&s.bad_output[first >> 5], bad_output << (first & 31));
        }
        if (i == j) {
#pragma unroll
          for (int c = 0; c < 4; ++c) s.own[i].at(r, 4 * g + c) = x[c];
        } else {
          store_operand(s.step + step_at(i, j), (j | 1) < i, (j & 1) != 0, lane, x);
        }
        store_operand(s.read + read_at(i, j), (j | 1) <= i, (j & 1) != 0, lane, y);
      }
    }
    exchange();
    state_products();
    exchange();
  }

  const uint64_t bad_outputs = static_cast<uint64_t>(s.bad_output[1]) << 32 | s.bad_output[0];
  // Nodes that are bad, or whose u is in this column.
  uint64_t bad = static_cast<uint64_t>(s.bad_node[1]) << 32 | s.bad_node[0];
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  Pair u[(kTiles + 1) / 2];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    if (i >= tiles) break;
    const int first = 16 * i + 4 * g;
    const f32x4 see = load4(&s.seen[first]), look = load4(&s.look[first]);
    const f32x4 b = load4(&s.strength[first]);
    const f32x4 values = value_columns(v[i], lane);
    f32x4 x, out;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      x[c] = fmaf(see[c], seen[i][c], b[c] * values[c]);
      out[c] = look[c] * read[i][c];
    }
#pragma unroll
    for (int j = 0; j < i; j += 2) {
      const uint2* const step = s.step + step_at(i, j);
      x = j + 1 < i ? add_pair(step, lane, u[j / 2], x)
          : i < 2   ? add_single(step, lane, u[j / 2], x)
                    : x + add_single(step, lane, u[j / 2], zero);
    }
    bad |= static_cast<uint64_t>(solve(s.inverse[i], s.own[i], lane, x)) << (16 * i);
    uint2 part[3];
    split3_half(x, part);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      uint4& whole = u[i / 2][p];
      if (i % 2 == 0) whole.x = part[p].x, whole.y = part[p].y;
      else whole.z = part[p].x, whole.w = part[p].y;
    }
#pragma unroll
    for (int j = 0; j <= i; j += 2) {
      const uint2* const looked = s.read + read_at(i, j);
      out = j + 1 <= i ? add_pair(looked, lane, u[j / 2], out)
            : i < 2    ? add_single(looked, lane, u[j / 2], out)
                       : out + add_single(looked, lane, u[j / 2], zero);
    }
    if (__any(bad != 0) || bad_outputs != 0) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint64_t self = 1ull << (first + c);
        if ((bad & (s.above[first + c] | self)) | (bad_outputs & self)) {
          out[c] = __uint_as_float(0x7FC00000u);
        }
      }
    }
    // A node's outputs side by side, in pieces of 16 bytes as the keys were.
    const uint2 packed = transpose_quad(
        make_uint2(bf16_pair(out[0], out[1]), bf16_pair(out[2], out[3])), lane);
    const int node = first + (r & 3);
    const int at = 2 * wave + (r >> 3);  // piece
    reinterpret_cast<uint2*>(&s.out[16 * node + (at ^ (node & 15))])[r >> 2 & 1] = packed;
  }
  exchange();
  bf16_bits* const outputs = a.outputs + (begin * a.value_heads + h) * kDim;
  for (int p = threadIdx.x; p < 16 * nodes; p += kThreads) {
    const int node = p >> 4, at = p & 15;
    *reinterpret_cast<uint4*>(reinterpret_cast<char*>(outputs) +
                              (node * a.value_heads * kDim + 8 * at) * 2u) =
        s.out[16 * node + (at ^ (node & 15))];
  }
}

// ------------------------------------------------------------------ the commit

struct CommitShared {
  uint4 k[kMaxNodes * 16];  // the path's, like all that follows
  uint4 columns[kMaxNodes / 32][8][64];  // of k, a key a lane, for each 32 and accumulator
  Block inverse[kMaxNodes / 16];  // of each 16: -A^T, then N
  alignas(16) int32_t steep[kWaves];  // whether a cell of what each wavefront forms of A
                                      // and N is out of range
  alignas(16) uint2 step[kMaxNodes / 32][kBlockPlaces];  // -A of each 32's second 16 and first
  float k_square[kMaxNodes], k_unit[kMaxNodes];
  // Factors of a node: -b exp(G) / |k| of S k, b, and what carries u to the end of its 32.
  float seen[kMaxNodes], strength[kMaxNodes], weight[kMaxNodes];
  float sum[kMaxNodes], rest[kMaxNodes];  // G / ln 2 from the start of each 32
  float log_decay[kMaxNodes];
  int path[kMaxNodes];
};

// Two bf16 values held in fp32.
__device__ __forceinline__ uint32_t held_pair(float low, float high) {
  return upper_halves(__float_as_uint(low), __float_as_uint(high));
}

// A lane's row of a slice as eight accumulators of four keys: accumulator m holds run
// `run(m, place)` of four (place: the lane group, or a quad's number where the tile's 16 keys
// are an operand's rows).  Loads cover 64 bytes of a row each; for the stores the quads of
// lanes that hold neighbouring rows exchange their runs, so that each store instruction covers
// four rows of 256 bytes: of 256 states of 32 heads that alone takes 176 us, in runs of 64
// bytes 196, or with the nontemporal hint 226.
template <typename Pool>
struct StateRows;

template <>
struct StateRows<float> {
  static __device__ __forceinline__ int run(int m, int place) { return 4 * m + place; }
  static __device__ __forceinline__ void load(const float* slice, int r, int g, f32x4 (&x)[8]) {
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      x[m] = __builtin_nontemporal_load(
          reinterpret_cast<const f32x4*>(slice + r * kDim + 4 * run(m, g)));
    }
  }
  static __device__ __forceinline__ void store(float* slice, int lane, const f32x4 (&x)[8]) {
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int m = 0; m < 8; m += 4) {
      f32x4 row[4];  // of the quad's rows, run m + its place
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const f32x4 t = transpose_quad(
            f32x4{x[m][c], x[m + 1][c], x[m + 2][c], x[m + 3][c]}, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) row[i][c] = t[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __builtin_nontemporal_store(
            row[i], reinterpret_cast<f32x4*>(slice + ((r & 12) + i) * kDim +
                                             4 * run(m + (r & 3), g)));
      }
    }
  }
};

template <>
struct StateRows<bf16_bits> {
  static __device__ __forceinline__ int run(int m, int place) {
    return 8 * (m >> 1) + 2 * place + (m & 1);
  }
  static __device__ __forceinline__ void load(const bf16_bits* slice, int r, int g,
                                              f32x4 (&x)[8]) {
#pragma unroll
    for (int m = 0; m < 8; m += 2) {
      float w[8];
      widen8(stream_load(reinterpret_cast<const uint4*>(slice + r * kDim + 4 * run(m, g))), w);
      x[m] = f32x4{w[0], w[1], w[2], w[3]};
      x[m + 1] = f32x4{w[4], w[5], w[6], w[7]};
    }
  }
  // The pool's own type: one rounding a path.
  static __device__ __forceinline__ void store(bf16_bits* slice, int lane,
                                               const f32x4 (&x)[8]) {
    const int r = lane & 15, g = lane >> 4;
    u32x4_t row[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {  // a word of each of a lane's four 16-byte pieces
      f32x4 t;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4& of = x[2 * i + (c >> 1)];
        t[i] = __uint_as_float(c & 1 ? bf16_pair(of[2], of[3]) : bf16_pair(of[0], of[1]));
      }
      t = transpose_quad(t, lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) row[i][c] = __float_as_uint(t[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __builtin_nontemporal_store(
          row[i], reinterpret_cast<u32x4_t*>(slice + ((r & 12) + i) * kDim +
                                             4 * run(2 * (r & 3), g)));
    }
  }
};

// Run `run` of four keys of a staged row.
__device__ __forceinline__ uint2 staged_run(const uint4* rows, int row, int run) {
  return reinterpret_cast<const uint2*>(rows)[32 * row + ((run >> 1 ^ (row & 15)) << 1) +
                                              (run & 1)];
}

// A wavefront's 16 rows after the path, token by token: S <- e^g S + b (v - e^g S k) k^T.
// For paths whose inverses pass fp32's range, which their writes need not.  Its keys are read
// where they are used, a run at a time, so that it takes no more registers than the other form.
template <typename Pool>
__device__ __forceinline__ void commit_by_steps(const CommitShared& s, const DraftArgs& a,
                                                const bf16_bits* values, int length, int lane,
                                                f32x4 (&x)[8]) {
  const int r = lane & 15, g = lane >> 4;
#pragma unroll 1
  for (int node = 0; node < length; ++node) {
    const float log_decay = s.log_decay[node], unit = s.k_unit[node], b = s.strength[node];
    const float value = widen(values[s.path[node] * a.value_stride + r]);
    const float decay =
        decay_between(log_decay * static_cast<float>(kInverseLn2), 0.0f, 0.0f, 0.0f);
    auto key = [&](int m) {
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
      const uint2 w = staged_run(s.k, node, StateRows<Pool>::run(m, g));
      return f32x4{widen_low(w.x), widen_high(w.x), widen_low(w.y), widen_high(w.y)};
    };
    float seen = 0.0f;
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const f32x4 k = key(m);
      x[m] *= decay;
#pragma unroll
      for (int c = 0; c < 4; ++c) seen = fmaf(x[m][c], k[c], seen);
    }
    seen += __shfl_xor(seen, 16);
    seen += __shfl_xor(seen, 32);
    const float write = b * (value - unit * seen) * unit;
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const f32x4 k = key(m);
#pragma unroll
      for (int c = 0; c < 4; ++c) x[m][c] = fmaf(write, k[c], x[m][c]);
    }
  }
}

// A wavefront's 16 rows of the state stay in registers while the path's nodes are applied 32
// at a time, both as the products' operand and as the update's accumulators.  What depends
// on no state comes first (the path, its keys in LDS, for each 32 the inverses of A's two
// diagonal blocks and the block below them, by a wavefront each), so that nothing waits for
// another wavefront between one 32 and the next.
//
// What bounds it (32 heads): 256 paths of up to 16 nodes on an fp32 pool take 180 us, HBM
// (the state's reads and writes alone 176, 5.6 TB/s); 128 paths of up to 64 on a bf16 pool
// 99, where the bytes are 56: vector instructions and the waits of one chain, with three
// workgroups a compute unit.  16 nodes at a time, with no block below the diagonal but twice
// as many splits of the state, they take 114.
//
// Three workgroups a compute unit: 80 registers, which the compiler is held to for a bf16 pool
// (it takes 82 otherwise: 115 us).  An fp32 pool's form has 80 by itself; held to them it is
// ordered otherwise, and 256 paths take 186 us.
template <typename Pool>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(sizeof(Pool) == 2 ? 6 : 2)))
void commit_kernel(DraftArgs a) {
  typedef StateRows<Pool> Rows;
  constexpr int kPasses = kMaxNodes * 16 / kThreads;
  __shared__ CommitShared s;

  int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t head = static_cast<uint32_t>(xcd_contiguous_item(blockIdx.x, gridDim.x));
  const uint32_t n = head / a.value_heads, h = head % a.value_heads, hk = h / a.group;
  int32_t slot;
  uint64_t begin;
  const int nodes = request_nodes(a, n, slot, begin);
  const int last = uniform(a.accepted[n]);
  if (last < 0 || last >= nodes) return;

  // Every wavefront finds the path; the first one forms its tables.
  int parent = -1;
  float log_decay = 0.0f, strength = 0.0f;
  if (lane < nodes) parent = (a.parents + begin)[lane];
  if (wave == 0 && lane < nodes) {
    const uint64_t first = begin * a.value_heads + h;
    log_decay = (a.log_decay + first)[lane * a.value_heads];
    strength = widen((a.beta + first)[lane * a.value_heads]);
  }
  const int first_row = 16 * wave;
  Pool* const state = static_cast<Pool*>(a.pool) +
                      (static_cast<uint64_t>(slot) * a.value_heads + h) * kTile +
                      first_row * kDim;
  f32x4 cells[8];
  Rows::load(state, r, g, cells);

  if (parent >= lane) parent = -1;
  uint64_t on_path = 0;
  for (int node = last; node >= 0; node = __builtin_amdgcn_readlane(parent, node)) {
    on_path |= 1ull << node;
  }
  int length = __popcll(on_path);
  if (wave == 0) {
    if (lane >= length) {
      s.path[lane] = -1;
      s.strength[lane] = 0.0f;
      s.log_decay[lane] = 0.0f;
    }
    if (on_path >> lane & 1) {
      const int place = __popcll(on_path & ((1ull << lane) - 1));
      s.path[place] = lane;
      s.strength[place] = strength;
      s.log_decay[place] = log_decay;
    }
    wave_sync();
    const float own = s.log_decay[lane];  // a NaN stays: it is on the path
    double sum = own < static_cast<float>(kLeastLogDecay) ? kLeastLogDecay : own;
#pragma unroll
    for (int reach = 1; reach < 32; reach <<= 1) {
      const double before = __shfl_up(sum, reach);
      if ((lane & 31) >= reach) sum += before;
    }
    sum *= kInverseLn2;
    const float high = static_cast<float>(sum);
    s.sum[lane] = high;
    s.rest[lane] = static_cast<float>(sum - high);
  }
  exchange();

  const bf16_bits* const keys = a.keys + begin * a.key_stride + hk * kDim;
  const bf16_bits* const values = a.values + begin * a.value_stride + h * kDim + first_row;
  // Four of a lane's columns of the value of node 4 g + (r & 3) of the 16 from `at` on.
  auto value_of = [&](int at) {
    return *static_cast<const uint2*>(row_at(values, s.path[min(at + 4 * g + (r & 3), length - 1)],
                                             static_cast<uint32_t>(a.value_stride), r & 12));
  };
  {
    uint4 pieces[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int first = p * (kThreads / 16) + 4 * wave;
      pieces[p] = make_uint4(0, 0, 0, 0);
      if (first < length) {  // the same for a wavefront; rows past the path are its last
        pieces[p] = *static_cast<const uint4*>(
            row_at(keys, s.path[min(first + g, length - 1)], static_cast<uint32_t>(a.key_stride),
                   8 * r));
      }
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int first = p * (kThreads / 16) + 4 * wave;
      if (first < (length + 15) / 16 * 16) {
        const float square = stage_piece(s.k, first + g, r, pieces[p]);
        if (r == 0) s.k_square[first + g] = square;
      }
    }
  }
  uint2 v[2] = {value_of(0), value_of(16)};
  exchange();

  auto unit_of = [&](float square) { return a.normalize ? 1.0f / sqrtf(square + kUnitEps) : 1.0f; };
  int32_t steep = 0;
  if (16 * wave < length) {
    const int at = 16 * wave;
    f32x4 kk = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const uint4 k = staged(s.k, at + r, 4 * step + g);
      kk = mfma(k, k, kk);
    }
    const float unit_c = unit_of(s.k_square[at + r]);
    if (g == 0) {
      const int node = at + r, end = min(node | 31, length - 1);
      const float decay = decay_between(s.sum[node], s.rest[node], 0.0f, 0.0f);
      const float carry = decay_between(s.sum[end], s.rest[end], s.sum[node], s.rest[node]);
      s.k_unit[node] = unit_c;
      s.seen[node] = -s.strength[node] * (decay * unit_c);
      s.weight[node] = node < length ? carry * unit_c : 0.0f;
    }
    wave_sync();
    const f32x4 sum = load4(&s.sum[at + 4 * g]), rest = load4(&s.rest[at + 4 * g]);
    const f32x4 b = load4(&s.strength[at + 4 * g]), k_unit = load4(&s.k_unit[at + 4 * g]);
    const float sum_c = s.sum[at + r], rest_c = s.rest[at + r];
    Block& block = s.inverse[at / 16];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float decay = decay_between(sum[c], rest[c], sum_c, rest_c);
      const bool up = 4 * g + c > r && at + 4 * g + c < length;
      block.at(r, 4 * g + c) = up ? -b[c] * decay * (k_unit[c] * unit_c * kk[c]) : 0.0f;
    }
    wave_sync();
    steep = __any(!invert(block, block, r, g == 0));
  } else if (wave >= kWaves - 2 && 32 * (kWaves - 1 - wave) + 16 < length) {
    const int column = 32 * (kWaves - 1 - wave), row = column + 16;
    f32x4 kk = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      kk = mfma(staged(s.k, row + r, 4 * step + g), staged(s.k, column + r, 4 * step + g), kk);
    }
    const f32x4 sum = load4(&s.sum[row + 4 * g]), rest = load4(&s.rest[row + 4 * g]);
    const f32x4 b = load4(&s.strength[row + 4 * g]), square = load4(&s.k_square[row + 4 * g]);
    const float sum_c = s.sum[column + r], rest_c = s.rest[column + r];
    const float unit_c = unit_of(s.k_square[column + r]);
    f32x4 x;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float decay = decay_between(sum[c], rest[c], sum_c, rest_c);
      const float k_unit = unit_of(square[c]);
      x[c] = row + 4 * g + c < length ? -b[c] * decay * (k_unit * unit_c * kk[c]) : 0.0f;
    }
    steep = __any(!in_range(x));
    store_operand(s.step[kWaves - 1 - wave], false, false, lane, x);
  }
  if (lane == 0) s.steep[wave] = steep;
  for (int at = 0; at < length; at += 32) {
    // Four keys of four nodes, a node a lane of a quad, to a key a lane.
    const int run = Rows::run(wave, r >> 2), row = 4 * g + (r & 3);
    const uint2 x = transpose_quad(staged_run(s.k + 16 * at, row, run), lane);
    uint2 y = make_uint2(0, 0);
    if (at + 16 < length) y = transpose_quad(staged_run(s.k + 16 * (at + 16), row, run), lane);
    s.columns[at / 32][wave][lane] = make_uint4(x.x, x.y, y.x, y.y);
  }
  exchange();

  if (__any(s.steep[lane % kWaves])) {
    asm volatile("" : "+v"(lane));
    commit_by_steps<Pool>(s, a, values, length, lane, cells);
    length = 0;
  }
  for (int at = 0; at < length; at += 32) {
    // Addresses by lane are formed in each round: kept over it, they take as many registers
    // as the state.
    asm volatile("" : "+v"(lane));
    r = lane & 15, g = lane >> 4;
    const bool two = at + 16 < length;
    f32x4 seen[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
    auto see = [&](const auto& part, int step) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i == 1 && !two) break;
        const uint4* const rows = s.k + 16 * (at + 16 * i);
        const uint2 low = staged_run(rows, r, Rows::run(2 * step, g));
        const uint2 high = staged_run(rows, r, Rows::run(2 * step + 1, g));
        seen[i] = product(make_uint4(low.x, low.y, high.x, high.y), part, seen[i]);
      }
    };
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const f32x4 x = cells[2 * step], y = cells[2 * step + 1];
      if (sizeof(Pool) == 2 && at == 0) {  // what was read has one part
        const uint4 part[1] = {make_uint4(held_pair(x[0], x[1]), held_pair(x[2], x[3]),
                                          held_pair(y[0], y[1]), held_pair(y[2], y[3]))};
        see(part, step);
      } else {
        uint4 part[3];
        split3(x, y, part);
        see(part, step);
      }
    }
    const int end = min(at + 31, length - 1);
    const float whole = decay_between(s.sum[end], s.rest[end], 0.0f, 0.0f);
    // Zeros where there is no second 16.
    uint4 part[3] = {};  // u, weighted: the first 16's and the second's side by side
    Pair first = {};     // u of the first 16
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && !two) break;
      const int node = at + 16 * i + 4 * g;
      const f32x4 own = value_columns(v[i], lane);
      if (at + 32 + 16 * i < length) v[i] = value_of(at + 32 + 16 * i);
      const f32x4 factor = load4(&s.seen[node]), b = load4(&s.strength[node]);
      f32x4 x;
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = fmaf(factor[c], seen[i][c], b[c] * own[c]);
      if (i == 1) x = add_single(s.step[at / 32], lane, first, x);
      const f32x4 u = block_product(s.inverse[at / 16 + i].run(r, 4 * g), x, x);
      uint2 half[3];
      if (i == 0 && two) {
        split3_half(u, half);
#pragma unroll
        for (int p = 0; p < 3; ++p) first[p].x = half[p].x, first[p].y = half[p].y;
      }
      split3_half(u * load4(&s.weight[node]), half);
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        if (i == 0) part[p].x = half[p].x, part[p].y = half[p].y;
        else part[p].z = half[p].x, part[p].w = half[p].y;
      }
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const uint4 key = s.columns[at / 32][m][lane];
      f32x4 x = cells[m] * whole;
#pragma unroll
      for (int p = 2; p >= 0; --p) x = mfma(key, part[p], x);
      cells[m] = x;
    }
  }
  Rows::store(state, lane, cells);
}

// ---------------------------------------------------------------------- launch

// 64 rows of it are 2^31 bytes, which the kernels' 32-bit offsets hold.
constexpr uint64_t kMaxStride = 1u << 24;  // elements between tokens

// By the most nodes that a tree may have, since lengths stay on the device: LDS and registers
// of the smaller forms let more workgroups share a compute unit (three, two and two on an fp32
// pool, four, four and two on a bf16 one).  Trees of 16 nodes, 32 heads, by the forms of 16, 32
// and 64: 256 on an fp32 pool 127, 129 and 134 us, on a bf16 pool 74, 74 and 92; 64 of them 31.8,
// 33.9 and 35.5, and 21.3, 21.4 and 26.2.  256 trees of up to 32 nodes by those of 32 and 64: 139
// and 142, and 81 and 102.
template <typename Pool>
int32_t launch_tree(void* stream, const DraftArgs& args, dim3 grid) {
  const uint32_t most = args.max_nodes < args.tokens ? args.max_nodes : args.tokens;
  const auto kernel = most <= 16   ? tree_kernel<Pool, 1>
                      : most <= 32 ? tree_kernel<Pool, 2>
                                   : tree_kernel<Pool, 4>;
  return launch(kernel, grid, dim3(kThreads), stream, args);
}

template <bool kCommit>
int32_t launch_drafts(void* stream, const gdn_state_codec_drafts* d, const int32_t* accepted,
                      void* pool, uint32_t slots, uint32_t pool_dtype, uint16_t* outputs) {
  if (!d || !pool || slots == 0 || slots > 0x7FFFFFFFu || pool_dtype > kDtypeBF16 ||
      d->requests == 0 || d->requests > GDN_STATE_CODEC_MAX_REQUESTS ||
      d->tokens > 0x7FFFFFFFu || d->key_heads == 0 || d->value_heads == 0 ||
      d->value_heads % d->key_heads != 0 || d->max_nodes == 0 || d->max_nodes > kMaxNodes ||
      d->normalize > 1 || d->query_stride % 8 != 0 || d->key_stride % 8 != 0 ||
      d->value_stride % 8 != 0 || d->query_stride > kMaxStride || d->key_stride > kMaxStride ||
      d->value_stride > kMaxStride || d->value_heads > kMaxStride / kDim || !d->offsets ||
      !d->slot_ids ||
      !token_rows(d->tokens, d->keys, d->values, d->log_decay, d->beta, d->parents) ||
      (kCommit ? !accepted || d->queries != nullptr
               : !token_rows(d->tokens, d->queries, outputs)) ||
      reinterpret_cast<uintptr_t>(d->parents) % sizeof(int32_t) != 0 ||
      !element_aligned(d->log_decay, d->beta) ||
      !aligned16(d->queries, d->keys, d->values, d->offsets, d->slot_ids, accepted, pool,
                 outputs)) {
    return kStatusInvalidArgument;
  }
  const uint64_t heads = static_cast<uint64_t>(d->requests) * d->value_heads;
  if (heads > kMaxGrid / kThreads) return kStatusInvalidArgument;  // threads of the grid
  if (d->tokens == 0) return kStatusOk;  // every tree is empty
  const DraftArgs args{d->queries, d->keys, d->values, d->log_decay, d->beta, d->query_stride,
                       d->key_stride, d->value_stride, d->parents, d->offsets, d->slot_ids,
                       accepted, pool, outputs, d->tokens, slots, d->value_heads,
                       d->value_heads / d->key_heads, d->max_nodes, d->scale, d->normalize};
  const dim3 grid(static_cast<uint32_t>(heads));
  const bool f32 = pool_dtype == kDtypeF32;
  if (kCommit) {
    return launch(f32 ? commit_kernel<float> : commit_kernel<bf16_bits>, grid, dim3(kThreads),
                  stream, args);
  }
  return f32 ? launch_tree<float>(stream, args, grid) : launch_tree<bf16_bits>(stream, args, grid);
}

}  // namespace
}  // namespace gdn

extern "C" int32_t statecentric_gdn_state_codec_gated_delta_tree_launch_v1(
    void* stream, const gdn_state_codec_drafts* drafts, const void* pool, uint32_t slots,
    uint32_t pool_dtype, uint16_t* outputs) {
  return gdn::launch_drafts<false>(stream, drafts, nullptr, const_cast<void*>(pool), slots,
                                   pool_dtype, outputs);
}

extern "C" int32_t statecentric_gdn_state_codec_gated_delta_commit_launch_v1(
    void* stream, const gdn_state_codec_drafts* drafts, const int32_t* accepted, void* pool,
    uint32_t slots, uint32_t pool_dtype) {
  return gdn::launch_drafts<true>(stream, drafts, accepted, pool, slots, pool_dtype, nullptr);
}
