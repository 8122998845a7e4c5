// Gradients of the gated delta rule's chunked form (formulas of the forward pass,
// layouts and precision in delta_chunk.h).
//
// With dS1 the gradient of a chunk's end state, dO of its outputs:
//   V' = P^T dO + exp(G_63 - G) K dS1,   X = V' + N^T (b V'),   Y = b X (= dV),
//   dS0 = exp(G_63) dS1 + (exp(G) Q)^T dO - (exp(G) K)^T Y
// run chunk after chunk, the last first, a column of the state by itself
// (delta_back_scan_kernel, the mirror of the forward scan).  What is left needs no
// order and takes whole rows (delta_gradient_kernel): with U = b E,
//   F_ij = exp(G_i - G_j) dO_i.U_j (j <= i),   H_ij = exp(G_i - G_j) Y_i.U_j (j < i),
//   dq_i = exp(G_i) S0 dO_i + sum_j F_ij k_j
//   dk_i = - exp(G_i) S0 Y_i - sum_j H_ij k_j                     (as it is read)
//          + exp(G_63 - G_i) dS1 U_i + sum_j F_ji q_j - sum_j H_ji k_j  (as it is written)
//   db_i = X_i.E_i
//   dG_i = q_i.dq_i + k_i.(dk_i as read) - k_i.(dk_i as written),
//   dG_63 += exp(G_63) <dS1, S0> + sum_j k_j.(exp(G_63 - G_j) dS1 U_j)
// for unit k and scaled unit q; dg is the sum of dG from a token to the chunk's
// end, and the raw gradients follow through the norms.  A key head's gradients are
// summed over its value heads in registers, in order.
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

// A chunk's operands in LDS: K (16 tiles), K^T and Q^T (32), the factors (2 tiles,
// the second's end not used) and N^T (18).  P^T stays in registers: with it, two
// stages would not fit.
constexpr int kStageRows = 0;
constexpr int kStageColumns = kKeyTiles * kTileBytes;
constexpr int kStageFactors = 3 * kKeyTiles * kTileBytes;
constexpr int kStageSolve = kStageFactors + 2 * kTileBytes;
constexpr int kStageTiles = 3 * kKeyTiles + 2 + kSolveParts * kTriangle;
constexpr int kStage = kStageTiles * kTileBytes;
static_assert(kHeadFactors <= 2 * kTileBytes, "the factors' tiles");
static_assert(2 * kStage <= static_cast<int>(kLdsPerCu), "two stages fit the LDS");
constexpr int kWaves = 4;
static_assert(kStageTiles % kWaves == 0, "tiles deal out evenly");

__global__ __launch_bounds__(64 * kWaves, 1) void delta_back_scan_kernel(BackArgs args) {
  constexpr int kSlices = kDim / (16 * kWaves);
  __shared__ __align__(16) char stages[2][kStage];
  const RuleArgs& a = args.rule;
  const ChunkSpace& space = a.space;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const uint32_t turn = blockIdx.x >> 3;  // slices of a head on one XCD, as forward
  const uint64_t item = static_cast<uint64_t>(turn / kSlices) * 8 + (blockIdx.x & 7);
  if (item >= static_cast<uint64_t>(a.requests) * space.value_heads) return;
  const uint32_t head = static_cast<uint32_t>(item % space.value_heads);
  const int32_t request = a.order[item / space.value_heads];
  if (request < 0 || static_cast<uint32_t>(request) >= a.requests) return;
  const int value = (turn % kSlices) * 16 * kWaves + 16 * wave + r;
  const uint64_t tile = (static_cast<uint64_t>(request) * space.value_heads + head) * kTile +
                        value * kDim + 4 * g;

  f32x4 state[8];  // the state's gradient, keys 16 t + 4 g + i
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    state[t] = args.d_final ? load4(args.d_final + tile + 16 * t) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const uint32_t first_row = min(static_cast<uint32_t>(a.chunk_offsets[request]), space.rows);
  const uint32_t rows = min(static_cast<uint32_t>(a.chunk_offsets[request + 1]), space.rows) -
                        first_row;
  const uint32_t begin = min(static_cast<uint32_t>(a.offsets[request]), a.tokens);
  const uint32_t length = min(static_cast<uint32_t>(a.offsets[request + 1]), a.tokens) - begin;
  const uint32_t chunks = min(rows, (length + kChunk - 1) / kChunk);
  const uint32_t stage_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) char*)&stages[0][0]));
  const uint64_t token_step = static_cast<uint64_t>(space.value_heads) * kDim;

  bf16_bits outs[4][4];            // dO of the tokens 16 t + 4 g + i
  uint4 back[kSolveParts * kTriangle];  // P^T
  const auto fetch = [&](uint32_t c) {
    const char* const keys = space.key_block(first_row + c, head / a.group);
    const char* const block = space.value_block(first_row + c, head);
#pragma unroll
    for (int i = 0; i < kStageTiles / kWaves; ++i) {
      const int t = i * kWaves + wave;
      const char* from = t < 16   ? keys + kKeyRows + t * kTileBytes
                         : t < 48 ? keys + kKeyColumns + (t - 16) * kTileBytes
                         : t < 50 ? block + (t - 48) * kTileBytes
                                  : block + kSolveBack + (t - 50) * kTileBytes;
      stage_tile(from, lane, stage_at + (c & 1) * kStage + t * kTileBytes);
    }
    const uint4* const p = reinterpret_cast<const uint4*>(block + kReadBack) + lane;
#pragma unroll
    for (int i = 0; i < kSolveParts * kTriangle; ++i) back[i] = p[i * 64];
    const int last = min(static_cast<int>(length - c * kChunk), kChunk) - 1;
    const bf16_bits* d = args.d_outputs + (begin + c * kChunk) * token_step + head * kDim + value;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) outs[t][i] = d[min(16 * t + 4 * g + i, last) * token_step];
    }
  };
  if (chunks != 0) fetch(chunks - 1);

  f32x4 x[4], y[4];
  const auto store_rows = [&](uint32_t c, int tokens) {
    float* e = space.error_gradient(first_row + c, head) + value;
    bf16_bits* d = args.d_values + (begin + c * kChunk) * token_step + head * kDim + value;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int token = 16 * t + 4 * g + i;
        e[token * kDim] = x[t][i];
        if (token < tokens) {
          d[token * token_step] = static_cast<bf16_bits>(bf16_pair(y[t][i], 0.0f));
        }
      }
    }
  };

  for (uint32_t c = chunks; c-- > 0;) {
    stage_ready();
    const uint32_t row = first_row + c;
    const char* const stage = stages[c & 1];
    const uint4* const k_rows = reinterpret_cast<const uint4*>(stage + kStageRows) + lane;
    const uint4* const k_columns = reinterpret_cast<const uint4*>(stage + kStageColumns) + lane;
    const uint4* const q_columns = k_columns + kKeyTiles * 64;
    const uint4* const solve = reinterpret_cast<const uint4*>(stage + kStageSolve) + lane;
    const float* const factors = reinterpret_cast<const float*>(stage + kStageFactors) + 4 * g;
    const int tokens = min(static_cast<int>(length - c * kChunk), kChunk);
    // Used before the next loads are issued, so that no wait for these covers them.
    uint32_t d_out[4][4];
    uint4 read_back[kSolveParts * kTriangle];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d_out[t][i] = 16 * t + 4 * g + i < tokens ? outs[t][i] : 0;
        asm volatile("" : "+v"(d_out[t][i]));
      }
    }
#pragma unroll
    for (int i = 0; i < kSolveParts * kTriangle; ++i) {
      read_back[i] = back[i];
      asm volatile("" : "+v"(read_back[i].x), "+v"(read_back[i].y), "+v"(read_back[i].z),
                   "+v"(read_back[i].w));
    }
    // V' of P^T dO, which needs no state; then P^T's registers take the next chunk's.
    f32x4 v[4];
    uint4 d_part[2];
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      d_part[step] = make_uint4(d_out[2 * step][0] | d_out[2 * step][1] << 16,
                                d_out[2 * step][2] | d_out[2 * step][3] << 16,
                                d_out[2 * step + 1][0] | d_out[2 * step + 1][1] << 16,
                                d_out[2 * step + 1][2] | d_out[2 * step + 1][3] << 16);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      v[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int step = upper_first(t); step < 2; ++step) {
        uint4 p[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) p[i] = read_back[i * kTriangle + upper_tile(t, step)];
        v[t] = mfma3(p, d_part[step], v[t]);
      }
    }
    if (c != 0) fetch(c - 1);
    if (c + 1 != chunks) {
      store_rows(c + 1, min(static_cast<int>(length - (c + 1) * kChunk), kChunk));
    }
    {
      float* p = space.state_gradient(row, head) + value;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[(16 * t + 4 * g + i) * kDim] = state[t][i];
      }
    }
    {
      uint4 part[4][3];
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        split3(state[2 * step], state[2 * step + 1], part[step]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 seen = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          seen = mfma3(k_rows[(4 * t + step) * 64], part[step], seen);
        }
        const f32x4 factor = load4(factors + kWrite * kChunk + 16 * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[t][i] = fmaf(factor[i], seen[i], v[t][i]);
      }
    }
    // X = V' + N^T (b V')
    {
      uint4 part[2][3];
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        f32x4 w[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x4 b = load4(factors + kStrength * kChunk + 32 * step + 16 * u);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[u][i] = b[i] * v[2 * step + u][i];
        }
        split3(w[0], w[1], part[step]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        x[t] = v[t];
#pragma unroll
        for (int step = upper_first(t); step < 2; ++step) {
          uint4 n[3];
#pragma unroll
          for (int p = 0; p < 3; ++p) n[p] = solve[(p * kTriangle + upper_tile(t, step)) * 64];
          x[t] = mfma6(n, part[step], x[t]);
        }
        const f32x4 b = load4(factors + kStrength * kChunk + 16 * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[t][i] = b[i] * x[t][i];
      }
    }
    // dS0
    const float whole = factors[kWhole * kChunk];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) state[t][i] *= whole;
    }
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      uint4 by_query[3], by_key[3];
      f32x4 p[2], m[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f32x4 q = load4(factors + kReadQuery * kChunk + 32 * step + 16 * u);
        const f32x4 k = load4(factors + kReadKey * kChunk + 32 * step + 16 * u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[u][i] = q[i] * widen_low(d_out[2 * step + u][i]);
          m[u][i] = -k[i] * y[2 * step + u][i];
        }
      }
      split3(p[0], p[1], by_query);
      split3(m[0], m[1], by_key);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        state[t] = mfma3(q_columns[(2 * t + step) * 64], by_query, state[t]);
        state[t] = mfma3(k_columns[(2 * t + step) * 64], by_key, state[t]);
      }
    }
  }
  if (chunks != 0) store_rows(0, min(static_cast<int>(length), kChunk));

  if (args.d_initial) {
#pragma unroll
    for (int t = 0; t < 8; ++t) store_cells(args.d_initial + tile + 16 * t, state[t]);
  }
}

// ------------------------------------------------------- q, k, g and b

constexpr int kThreads = 256;
constexpr int kWide = 68;  // fp32 a row of a 64 x 64 matrix

// Eight neighbouring values of a row, as an operand's places of natural order.
__device__ __forceinline__ void split_row(const float* p, uint4 (&part)[3]) {
  split3(load4(p), load4(p + 4), part);
}

__device__ __forceinline__ float sum16(float x) {  // over the 16 lanes of a DPP row
  x = add_partner<1>(x);
  x = add_partner<2>(x);
  x = add_partner<4>(x);
  return add_partner<8>(x);
}

// One workgroup per chunk row and key head; wavefront w takes keys 32 w..32 w + 31
// of all 64 tokens, and token rows 16 w.. of F and H.
__global__ __launch_bounds__(kThreads, 1) void delta_gradient_kernel(BackArgs args) {
  __shared__ __align__(16) float f[kChunk][kWide];
  __shared__ __align__(16) float h[kChunk][kWide];
  __shared__ __align__(16) float factors[kFactors][kChunk];
  __shared__ __align__(16) float norms[3][kChunk];  // 1/|k|, scale/|q|, 1/|q|
  __shared__ float sums[3][4][kChunk];
  __shared__ float ends[4];
  const RuleArgs& a = args.rule;
  const ChunkSpace& space = a.space;
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63, r = lane & 15, g = lane >> 4;
  const uint32_t row = blockIdx.x / space.key_heads;
  const uint32_t head = blockIdx.x % space.key_heads;
  const uint64_t token_step = static_cast<uint64_t>(space.value_heads) * kDim;
  if (row == 0) {  // tokens of no request: zeros
    const uint32_t from = min(static_cast<uint32_t>(a.offsets[a.requests]), a.tokens);
    for (uint64_t token = from; token < a.tokens; ++token) {
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
  const int key = 32 * wave + r;  // and 16 more

  // This wavefront's columns of q and k, as operands over tokens and as they meet
  // an accumulator (token 16 i + 4 g + j).
  uint4 k_columns[2][2], q_columns[2][2];
  float k_cells[2][4][4], q_cells[2][4][4];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      const int at = (2 * (2 * wave + c) + step) * kTileBytes + 16 * lane;
      const uint4 k = *reinterpret_cast<const uint4*>(keys + kKeyColumns + at);
      const uint4 q = *reinterpret_cast<const uint4*>(keys + kQueryColumns + at);
      k_columns[c][step] = k, q_columns[c][step] = q;
      float kx[8], qx[8];
      widen8(k, kx);
      widen8(q, qx);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        k_cells[c][2 * step + j / 4][j % 4] = kx[j];
        q_cells[c][2 * step + j / 4][j % 4] = qx[j];
      }
    }
  }
  if (t < 3 * kChunk) {
    norms[t / kChunk][t % kChunk] = reinterpret_cast<const float*>(keys + kNorms)[t];
  }

  f32x4 d_q[2][4] = {}, d_k[2][4] = {};
  for (uint32_t member = 0; member < a.group; ++member) {
    const uint32_t value_head = head * a.group + member;
    const float* const s0 = space.state(row, value_head);
    const float* const s1 = space.state_gradient(row, value_head);
    const float* const errors = space.errors(row, value_head);
    const float* const xs = space.error_gradient(row, value_head);
    const bf16_bits* const d_out = args.d_outputs + first * token_step + value_head * kDim;
    const auto d_row = [&](int token, int step) {  // dO as an operand over values
      return token < count ? *reinterpret_cast<const uint4*>(d_out + token * token_step +
                                                             32 * step + 8 * g)
                           : make_uint4(0, 0, 0, 0);
    };
    __syncthreads();  // the last head's f, h, factors and sums have been read
    for (int i = t; i < kFactors * kChunk; i += kThreads) {
      factors[i / kChunk][i % kChunk] =
          reinterpret_cast<const float*>(space.value_block(row, value_head))[i];
    }
    __syncthreads();

    {  // F and H, rows 16 wave + 4 g + j
      uint4 x_part[4][3], o_part[4];
      const int token = 16 * wave + r;
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        split_row(xs + token * kDim + 32 * step + 8 * g, x_part[step]);
        o_part[step] = d_row(token, step);
      }
      for (int c = 0; c < 4; ++c) {
        f32x4 fx = {0.0f, 0.0f, 0.0f, 0.0f}, hx = fx;
        if (c <= wave) {
          float along = 0.0f;
#pragma unroll
          for (int step = 0; step < 4; ++step) {
            const float* e = errors + (16 * c + r) * kDim + 32 * step + 8 * g;
            uint4 e_part[3];
            split_row(e, e_part);
            fx = mfma3(o_part[step], e_part, fx);
            hx = mfma6(x_part[step], e_part, hx);
            if (c == wave) {
              const float* x = xs + token * kDim + 32 * step + 8 * g;
#pragma unroll
              for (int j = 0; j < 8; ++j) along = fmaf(x[j], e[j], along);
            }
          }
          if (c == wave) {  // X.E of the token, over the four lane groups
            along = add_partner<32>(add_partner<16>(along));
            if (g == 0 && token < count) {
              args.d_beta[(first + token) * space.value_heads + value_head] =
                  static_cast<bf16_bits>(bf16_pair(along, 0.0f));
            }
          }
        }
        const int column = 16 * c + r;
        const float b_column = factors[kStrength][column];
        const float sum = factors[kSum][column], rest = factors[kSumRest][column];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 16 * wave + 4 * g + j;
          const float decay = expf((factors[kSum][i] - sum) + (factors[kSumRest][i] - rest));
          f[i][column] = column <= i ? decay * (fx[j] * b_column) : 0.0f;
          h[i][column] = column < i ? decay * (factors[kStrength][i] * hx[j] * b_column) : 0.0f;
        }
      }
    }

    // S0 dO, S0 X and dS1 E of this wavefront's keys.
    f32x4 read_q[2][4] = {}, read_k[2][4] = {}, written[2][4] = {};
    float end = 0.0f;
    {
      uint4 part[2][4][3];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          split_row(s0 + (key + 16 * c) * kDim + 32 * step + 8 * g, part[c][step]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          uint4 x_part[3];
          split_row(xs + (16 * i + r) * kDim + 32 * step + 8 * g, x_part);
          const uint4 o = d_row(16 * i + r, step);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            read_q[c][i] = mfma3(o, part[c][step], read_q[c][i]);
            read_k[c][i] = mfma6(x_part, part[c][step], read_k[c][i]);
          }
        }
      }
    }
    {
      uint4 part[2][4][3];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          const uint64_t at = (key + 16 * c) * kDim + 32 * step + 8 * g;
          const f32x4 x = load4(s1 + at), y = load4(s1 + at + 4);
          const f32x4 u = load4(s0 + at), v = load4(s0 + at + 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) end = fmaf(x[j], u[j], fmaf(y[j], v[j], end));
          split3(x, y, part[c][step]);
        }
      }
      end *= factors[kWhole][0];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          uint4 e_part[3];
          split_row(errors + (16 * i + r) * kDim + 32 * step + 8 * g, e_part);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            written[c][i] = mfma6(e_part, part[c][step], written[c][i]);
          }
        }
      }
    }
    __syncthreads();  // f and h are whole

    // The products with F and H and their transposes, row tile by row tile.
    float flux[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 b = load4(&factors[kStrength][16 * i + 4 * g]);
      f32x4 by_query[2], by_read[2], by_write[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        by_query[c] = by_read[c] = by_write[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        const int at = 32 * step + 4 * g;  // places at.. and at + 16..
        if (step < lower_steps(i)) {  // row token 16 i + r, over the tokens before it
          const f32x4 u = load4(&norms[0][at]), v = load4(&norms[0][at + 16]);
          f32x4 x = load4(&f[16 * i + r][at]), y = load4(&f[16 * i + r][at + 16]);
          uint4 part[3];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] *= u[j], y[j] *= v[j];
          split3(x, y, part);
#pragma unroll
          for (int c = 0; c < 2; ++c) by_query[c] = mfma3(part, k_columns[c][step], by_query[c]);
          x = load4(&h[16 * i + r][at]), y = load4(&h[16 * i + r][at + 16]);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] *= u[j], y[j] *= v[j];
          split3(x, y, part);
#pragma unroll
          for (int c = 0; c < 2; ++c) by_read[c] = mfma3(part, k_columns[c][step], by_read[c]);
        }
        if (step >= upper_first(i)) {  // row token 16 i + r, over the tokens after it
          f32x4 x, y;
          uint4 part[3];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[j] = f[at + j][16 * i + r] * norms[1][at + j];
            y[j] = f[at + 16 + j][16 * i + r] * norms[1][at + 16 + j];
          }
          split3(x, y, part);
#pragma unroll
          for (int c = 0; c < 2; ++c) by_write[c] = mfma3(part, q_columns[c][step], by_write[c]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[j] = -h[at + j][16 * i + r] * norms[0][at + j];
            y[j] = -h[at + 16 + j][16 * i + r] * norms[0][at + 16 + j];
          }
          split3(x, y, part);
#pragma unroll
          for (int c = 0; c < 2; ++c) by_write[c] = mfma3(part, k_columns[c][step], by_write[c]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int token = 16 * i + 4 * g + j;
        const float k_unit = norms[0][token], q_unit = norms[1][token];
        const float decay = expf(factors[kSum][token]);
        const float kept = expf((factors[kSum][kChunk - 1] - factors[kSum][token]) +
                                (factors[kSumRest][kChunk - 1] - factors[kSumRest][token]));
        float total = 0.0f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float dq = fmaf(decay, read_q[c][i][j], by_query[c][j]);
          const float read = -fmaf(decay * b[j], read_k[c][i][j], by_read[c][j]);
          const float carried = kept * b[j] * written[c][i][j];
          const float write = carried + by_write[c][j];
          const float k = k_unit * k_cells[c][i][j], q = q_unit * q_cells[c][i][j];
          total = fmaf(q, dq, fmaf(k, read - write, total));
          end = fmaf(k, carried, end);
          d_q[c][i][j] += dq;
          d_k[c][i][j] += read + write;
        }
        flux[i][j] = sum16(total);
      }
    }
    end = wave_sum_valu(end);
    if (lane == 0) ends[wave] = end;
    if (r == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[0][wave][16 * i + 4 * g + j] = flux[i][j];
      }
    }
    __syncthreads();
    if (wave == 0) {
      float total = (sums[0][0][lane] + sums[0][1][lane]) + (sums[0][2][lane] + sums[0][3][lane]);
      if (lane == 63) total += (ends[0] + ends[1]) + (ends[2] + ends[3]);
#pragma unroll
      for (int step = 1; step < 64; step <<= 1) {  // from each token to the chunk's end
        const float after = __shfl_down(total, step);
        if (lane + step < 64) total += after;
      }
      if (lane < count) {
        args.d_log_decay[(first + lane) * space.value_heads + value_head] = total;
      }
    }
  }

  // Through the norms: with u = scale / |q|, d(raw) = u dq - q (u q.dq) / |q|^2, and
  // for keys the same with scale 1.
  if (a.normalize) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float q = 0.0f, k = 0.0f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          q = fmaf(q_cells[c][i][j], d_q[c][i][j], q);
          k = fmaf(k_cells[c][i][j], d_k[c][i][j], k);
        }
        q = sum16(q), k = sum16(k);
        if (r == 0) {
          sums[1][wave][16 * i + 4 * g + j] = q;
          sums[2][wave][16 * i + 4 * g + j] = k;
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int token = 16 * i + 4 * g + j;
      const float k_unit = norms[0][token], q_unit = norms[1][token];
      float q_along = 0.0f, k_along = 0.0f;
      if (a.normalize) {
        q_along = ((sums[1][0][token] + sums[1][1][token]) +
                   (sums[1][2][token] + sums[1][3][token])) *
                  q_unit * norms[2][token] * norms[2][token];
        k_along = ((sums[2][0][token] + sums[2][1][token]) +
                   (sums[2][2][token] + sums[2][3][token])) *
                  k_unit * k_unit * k_unit;
      }
      if (token < count) {
        const uint64_t at = ((first + token) * space.key_heads + head) * kDim + key;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float dq = fmaf(-q_cells[c][i][j], q_along, q_unit * d_q[c][i][j]);
          const float dk = fmaf(-k_cells[c][i][j], k_along, k_unit * d_k[c][i][j]);
          args.d_queries[at + 16 * c] = static_cast<bf16_bits>(bf16_pair(dq, 0.0f));
          args.d_keys[at + 16 * c] = static_cast<bf16_bits>(bf16_pair(dk, 0.0f));
        }
      }
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
  if (!gdn::rule_args(rule, true, args.rule) || !d_outputs || !d_queries || !d_keys ||
      !d_values || !d_log_decay || !d_beta ||
      !gdn::aligned16(d_outputs, d_final, d_queries, d_keys, d_values, d_log_decay, d_beta,
                      d_initial)) {
    return gdn::kStatusInvalidArgument;
  }
  args.d_outputs = d_outputs, args.d_final = d_final, args.d_initial = d_initial;
  args.d_queries = d_queries, args.d_keys = d_keys, args.d_values = d_values;
  args.d_log_decay = d_log_decay, args.d_beta = d_beta;
  const gdn::ChunkSpace& space = args.rule.space;
  const uint64_t items = static_cast<uint64_t>(rule->requests) * rule->value_heads;
  const uint64_t scans = (items + 7) / 8 * 8 * (gdn::kDim / (16 * gdn::kWaves));
  if (scans > gdn::kMaxGrid) return gdn::kStatusInvalidArgument;
  const int32_t status = gdn::launch(gdn::delta_back_scan_kernel,
                                     dim3(static_cast<uint32_t>(scans)),
                                     dim3(64 * gdn::kWaves), stream, args);
  return status != gdn::kStatusOk
             ? status
             : gdn::launch(gdn::delta_gradient_kernel, dim3(space.rows * space.key_heads),
                           dim3(gdn::kThreads), stream, args);
}
