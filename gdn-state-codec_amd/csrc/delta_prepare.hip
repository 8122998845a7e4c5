// The state-independent half of the gated delta rule's chunked form, for every
// chunk and key head at once: the transposed operands, the norms, and for each
// value head of the group the factors, N b and P b (and for training N^T b and P^T);
// formulas and layouts in delta_chunk.h.
//
// One workgroup per chunk row and key head.  K K^T and Q K^T are formed once per
// key head on the matrix cores (exact bf16 products), then each wavefront takes a
// value head's N b or its P b, with no barrier between them.
//
// N by blocks of 16 tokens.  The four diagonal blocks are solved at once by forward
// substitution, one column a lane (120 fmas).  Below them
//   N_ij = -(I + N_ii b_i) (A_ij + sum_(j<=m<i) A_im b_m N_mj)
// is 16 products of 16 x 16 on the fp32 matrix cores, each block an accumulator
// that is the next product's operand as it is.  Substitution and this recursion
// are stable for any keys, which powers of A are not.
//
// Bound by what it writes: of 32,768 tokens, 16 key heads and 32 value heads it reads
// 268 MB and writes 671 in 200 us, 4.7 TB/s (a copy: 6.1; 220 us with the matrices whole
// and two workgroups a compute unit); a training pass of 5,298 tokens, with the
// transposes and the products of unit rows, takes 63 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "delta_chunk.h"
#include "lane_exchange.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr int kPitch = 136;  // bf16 a staged row: 128 and 16 bytes against bank conflicts
constexpr double kInverseLn2 = 1.4426950408889634074;

struct Head {  // one wavefront's value head
  float sum[kChunk], rest[kChunk];  // G / ln 2
  float strength[kChunk];
};

// A lower triangular 64 x 64 matrix: ten blocks of 16 x 16, and the two above the
// diagonal that an operand tile holds beside them.  A row's four runs of four columns
// are rotated by its place, so that 16 rows' runs fall on different banks.
struct Triangle {
  float cells[12][256];

  static __device__ __forceinline__ int block(int i, int j) {
    return j <= i ? i * (i + 1) / 2 + j : i == 0 ? 10 : 11;
  }
  // Four columns from `column` on (a multiple of 4), of row `row` of a block.
  __device__ __forceinline__ float* run(int at, int row, int column) {
    return &cells[at][16 * row + (column ^ (row & 12))];
  }
  __device__ __forceinline__ const float* run(int at, int row, int column) const {
    return &cells[at][16 * row + (column ^ (row & 12))];
  }
  __device__ __forceinline__ float& cell(int at, int row, int column) {
    return cells[at][16 * row + (column ^ (row & 12))];
  }
  __device__ __forceinline__ float cell(int at, int row, int column) const {
    return cells[at][16 * row + (column ^ (row & 12))];
  }
};

struct Staged {
  union {
    struct {
      uint16_t k[kChunk][kPitch];
      uint16_t q[kChunk][kPitch];
    };
    struct {
      Triangle kk, qk;
      Triangle solve[2];  // A, then N, of two wavefronts
    };
  };
  Head heads[4];
  float k_unit[kChunk];  // 1 / |k|
  float q_unit[kChunk];  // scale / |q|
  float q_norm[kChunk];  // 1 / |q|
};
static_assert(workgroups_by_lds(sizeof(Staged)) == 3, "three workgroups share a compute unit");

// LDS written by other lanes of the same wavefront is read after this.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// c + a b for 16 x 16 fp32 blocks: lane l has row l & 15, columns 4 g.. of a, and
// rows 4 g.. of b's column l & 15 (an accumulator).
__device__ __forceinline__ f32x4 block_product(const f32x4& a, const f32x4& b, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

__device__ __forceinline__ f32x4 times(const f32x4& a, const f32x4& b) {
  return f32x4{a[0] * b[0], a[1] * b[1], a[2] * b[2], a[3] * b[3]};
}

__device__ __forceinline__ void store_tile(char* operand, int tile, int lane, const f32x4& x,
                                           const f32x4& y) {
  uint4 part[3];
  split3(x, y, part);
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    reinterpret_cast<uint4*>(operand + (p * kTriangle + tile) * kTileBytes)[lane] = part[p];
  }
}

template <bool kTrain>
__device__ __forceinline__ void solve_head(Staged& s, const Head& head, Triangle& m, int lane,
                                           char* block) {
  const int r = lane & 15, g = lane >> 4;
  // A, block by block as accumulators (row 4 g + i, column r), and in LDS.
  f32x4 a[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 sum = load4(&head.sum[16 * i + 4 * g]), rest = load4(&head.rest[16 * i + 4 * g]);
    const f32x4 unit = load4(&s.k_unit[16 * i + 4 * g]);
#pragma unroll
    for (int j = 0; j <= i; ++j) {
      const int column = 16 * j + r;
      const float sum_c = head.sum[column], rest_c = head.rest[column];
      const float unit_c = s.k_unit[column];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int row = 16 * i + 4 * g + c;
        const float x = decay_between(sum[c], rest[c], sum_c, rest_c) *
                        (unit[c] * unit_c * s.kk.cell(Triangle::block(i, j), 4 * g + c, r));
        a[i][j][c] = column < row ? x : 0.0f;
        m.cell(Triangle::block(i, j), 4 * g + c, r) = a[i][j][c];
      }
    }
  }
  wave_sync();
  {  // the diagonal blocks: lane group g solves block g, column r
    float n[16], scaled[16];
    const float* const strength = &head.strength[16 * g];
    const int diagonal = g * (g + 3) / 2;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x = -m.cell(diagonal, i, r), y = 0.0f;
#pragma unroll
      for (int c = 0; c < i; c += 4) {
        const f32x4 l = load4(m.run(diagonal, i, c));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (c + u < i) {
            if (u & 1) y = fmaf(-l[u], scaled[c + u], y);
            else x = fmaf(-l[u], scaled[c + u], x);
          }
        }
      }
      n[i] = x + y;
      scaled[i] = strength[i] * n[i];
    }
    wave_sync();  // A's diagonal blocks have been read
#pragma unroll
    for (int i = 0; i < 16; ++i) m.cell(diagonal, i, r) = n[i];
  }
  wave_sync();
  f32x4 inverse[4];  // I + N_ii b_i, row r
  f32x4 n[4][4], scaled[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 row = load4(m.run(Triangle::block(i, i), r, 4 * g));
    const f32x4 b = load4(&head.strength[16 * i + 4 * g]);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      inverse[i][c] = fmaf(row[c], b[c], 4 * g + c == r ? 1.0f : 0.0f);
      n[i][i][c] = m.cell(Triangle::block(i, i), 4 * g + c, r);
    }
    scaled[i][i] = times(b, n[i][i]);
  }
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    const f32x4 b = load4(&head.strength[16 * i + 4 * g]);
#pragma unroll
    for (int j = 0; j < i; ++j) {
      f32x4 x = a[i][j];
#pragma unroll
      for (int c = j; c < i; ++c) {
        x = block_product(load4(m.run(Triangle::block(i, c), r, 4 * g)), scaled[c][j], x);
      }
      const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
      x = block_product(inverse[i], x, zero);
      n[i][j] = -x;
      scaled[i][j] = times(b, n[i][j]);
    }
  }
  wave_sync();  // A has been read
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool empty = (i == 0 && j == 1) || (i == 2 && j == 3);  // above, in a tile
      if (j < i || empty) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          m.cell(Triangle::block(i, j), 4 * g + c, r) = empty ? 0.0f : n[i][j][c];
        }
      }
    }
  }
  wave_sync();
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      if (step < lower_steps(t)) {
        const float* const b = &head.strength[32 * step + 4 * g];
        store_tile(block + kSolve, lower_tile(t, step), lane,
                   times(load4(m.run(Triangle::block(t, 2 * step), r, 4 * g)), load4(b)),
                   times(load4(m.run(Triangle::block(t, 2 * step + 1), r, 4 * g)), load4(b + 16)));
      }
      if (kTrain && step >= upper_first(t)) {
        f32x4 x, y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = m.cell(Triangle::block(2 * step, t), 4 * g + i, r);
          y[i] = m.cell(Triangle::block(2 * step + 1, t), 4 * g + i, r);
        }
        const float* const b = &head.strength[32 * step + 4 * g];
        store_tile(block + kSolveBack, upper_tile(t, step), lane, times(x, load4(b)),
                   times(y, load4(b + 16)));
      }
    }
  }
}

// P b of one value head (and P^T) by one wavefront.
template <bool kTrain>
__device__ __forceinline__ void read_out_head(const Staged& s, const Head& head, int lane,
                                              char* block) {
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int at = 16 * t + r;
    const float sum = head.sum[at], rest = head.rest[at];
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      f32x4 x[2];
      if (step < lower_steps(t)) {  // row i = at, columns j
        const float q_unit = s.q_unit[at];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int from = 32 * step + 16 * u + 4 * g;
          const f32x4 sums = load4(&head.sum[from]), rests = load4(&head.rest[from]);
          const f32x4 units = load4(&s.k_unit[from]), b = load4(&head.strength[from]);
          const f32x4 product = load4(s.qk.run(Triangle::block(t, 2 * step + u), r, 4 * g));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y = decay_between(sum, rest, sums[i], rests[i]) *
                            (q_unit * units[i] * product[i]) * b[i];
            x[u][i] = from + i <= at ? y : 0.0f;
          }
        }
        // Two parts, rounded: 2^-16 of a weight whose sums become bf16 outputs.
        uint4 high, low;
        split2_pair(x[0][0], x[0][1], high.x, low.x);
        split2_pair(x[0][2], x[0][3], high.y, low.y);
        split2_pair(x[1][0], x[1][1], high.z, low.z);
        split2_pair(x[1][2], x[1][3], high.w, low.w);
        uint4* const p = reinterpret_cast<uint4*>(block + kReadOut +
                                                  lower_tile(t, step) * kTileBytes) + lane;
        p[0] = high;
        p[kTriangle * 64] = low;
      }
      if (kTrain && step >= upper_first(t)) {  // row j = at, columns i
        const float k_unit = s.k_unit[at];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int from = 32 * step + 16 * u + 4 * g;
          const f32x4 sums = load4(&head.sum[from]), rests = load4(&head.rest[from]);
          const f32x4 units = load4(&s.q_unit[from]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y = decay_between(sums[i], rests[i], sum, rest) *
                            (units[i] * k_unit *
                             s.qk.cell(Triangle::block(2 * step + u, t), 4 * g + i, r));
            x[u][i] = at <= from + i ? y : 0.0f;
          }
        }
        store_tile(block + kReadBack, upper_tile(t, step), lane, x[0], x[1]);
      }
    }
  }
}

// The outputs of tokens of no request: zeros, for one key head's value heads, a share of
// the tokens for each chunk row.
__device__ __forceinline__ void clear_rest(const RuleArgs& a, uint32_t row, uint32_t head,
                                           bf16_bits* outputs) {
  const uint32_t from = min(static_cast<uint32_t>(a.offsets[a.requests]), a.tokens);
  const uint32_t width = a.group * kDim;
  for (uint64_t token = from + static_cast<uint64_t>(row); token < a.tokens;
       token += a.space.rows) {
    for (uint32_t i = threadIdx.x; i < width; i += kThreads) {
      outputs[token * a.space.value_heads * kDim + head * width + i] = 0;
    }
  }
}

// Three workgroups share a compute unit (training's registers allow two).
template <bool kTrain>
__global__ __launch_bounds__(kThreads, kTrain ? 2 : 3) void delta_prepare_kernel(RuleArgs a,
                                                                bf16_bits* outputs) {
  __shared__ __align__(16) Staged s;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t row = blockIdx.x / a.space.key_heads;
  const uint32_t head = blockIdx.x % a.space.key_heads;
  const int4 chunk = a.chunks[row];
  const int count = chunk_tokens(a, chunk);
  if (kTrain) clear_rest(a, row, head, outputs);
  if (count == 0 || (!kTrain && chunk.w < 0)) return;  // past the last chunk, or padding
  const uint64_t first = chunk.y;

  {  // stage the rows, 32 columns a thread, zeros past the request's end
    const int token = t >> 2, part = t & 3;
    uint4 k[4], q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k[i] = q[i] = make_uint4(0, 0, 0, 0);
      const int column = 32 * i + 8 * part;
      if (token < count) {
        k[i] = *reinterpret_cast<const uint4*>(a.keys + (first + token) * a.key_stride +
                                               head * kDim + column);
        q[i] = *reinterpret_cast<const uint4*>(a.queries + (first + token) * a.query_stride +
                                               head * kDim + column);
      }
    }
    float kk = 0.0f, qq = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int column = 32 * i + 8 * part;
      *reinterpret_cast<uint4*>(&s.k[token][column]) = k[i];
      *reinterpret_cast<uint4*>(&s.q[token][column]) = q[i];
      float x[8];
      widen8(k[i], x);
#pragma unroll
      for (int c = 0; c < 8; ++c) kk = fmaf(x[c], x[c], kk);
      widen8(q[i], x);
#pragma unroll
      for (int c = 0; c < 8; ++c) qq = fmaf(x[c], x[c], qq);
    }
    kk = add_partner<2>(add_partner<1>(kk));
    qq = add_partner<2>(add_partner<1>(qq));
    if (part == 0) {
      s.k_unit[token] = a.normalize ? 1.0f / sqrtf(kk + kUnitEps) : 1.0f;
      s.q_norm[token] = a.normalize ? 1.0f / sqrtf(qq + kUnitEps) : 1.0f;
      s.q_unit[token] = a.scale * s.q_norm[token];
    }
  }
  __syncthreads();

  char* const key_block = a.space.key_block(row, head);
  const int r = lane & 15, g = lane >> 4;
  f32x4 kk[4], qk[4];  // row tile `wave` of K K^T and Q K^T, up to the diagonal
  {
    uint4 k[4], q[4];
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      k[step] = *reinterpret_cast<const uint4*>(&s.k[16 * wave + r][32 * step + 8 * g]);
      q[step] = *reinterpret_cast<const uint4*>(&s.q[16 * wave + r][32 * step + 8 * g]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      kk[c] = qk[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (c <= wave) {
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          const uint4 b = *reinterpret_cast<const uint4*>(&s.k[16 * c + r][32 * step + 8 * g]);
          kk[c] = mfma(k[step], b, kk[c]);
          qk[c] = mfma(q[step], b, qk[c]);
        }
      }
    }
    // Two row tiles of the transposes: rows = keys in state order, over the tokens.
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int key = state_key(2 * wave + c, r);
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        uint32_t kw[4], qw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int x = token_place(step, g, 2 * i), y = token_place(step, g, 2 * i + 1);
          kw[i] = s.k[x][key] | static_cast<uint32_t>(s.k[y][key]) << 16;
          if constexpr (kTrain) qw[i] = s.q[x][key] | static_cast<uint32_t>(s.q[y][key]) << 16;
        }
        const int tile = (2 * (2 * wave + c) + step) * kTileBytes;
        reinterpret_cast<uint4*>(key_block + kKeyColumns + tile)[lane] =
            make_uint4(kw[0], kw[1], kw[2], kw[3]);
        if constexpr (kTrain) {
          reinterpret_cast<uint4*>(key_block + kQueryColumns + tile)[lane] =
              make_uint4(qw[0], qw[1], qw[2], qw[3]);
        }
      }
    }
    if (kTrain && t < kChunk) {
      float* norms = reinterpret_cast<float*>(key_block + kNorms);
      norms[t] = s.k_unit[t];
      norms[kChunk + t] = s.q_unit[t];
      norms[2 * kChunk + t] = s.q_norm[t];
    }
  }
  __syncthreads();  // K and Q have been read
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (c <= wave) {
      const int at = wave * (wave + 1) / 2 + c;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s.kk.cell(at, 4 * g + i, r) = kk[c][i];
        s.qk.cell(at, 4 * g + i, r) = qk[c][i];
      }
      if constexpr (kTrain) {  // of unit rows, for the decays' gradients
        const f32x4 k_unit = load4(&s.k_unit[16 * wave + 4 * g]);
        const f32x4 q_unit = load4(&s.q_unit[16 * wave + 4 * g]);
        const float unit = s.k_unit[16 * c + r];
        f32x4* const dots = reinterpret_cast<f32x4*>(key_block + kDots + 2 * at * kTileBytes);
        f32x4 x, y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = qk[c][i] * (q_unit[i] * unit);
          y[i] = kk[c][i] * (k_unit[i] * unit);
        }
        __builtin_nontemporal_store(x, dots + lane);  // read when both scans are done
        __builtin_nontemporal_store(y, dots + 64 + lane);
      }
    }
  }
  __syncthreads();

  // Wavefronts 0 and 2 solve, 1 and 3 form P b, each for every second value head.
  Head& mine = s.heads[wave];
  for (uint32_t member = wave >> 1; member < a.group; member += 2) {
    const uint32_t value_head = head * a.group + member;
    char* const block = a.space.value_block(row, value_head);
    const uint64_t at = (first + lane) * a.space.value_heads + value_head;
    // exp of anything below -10000 is 0; a sum of -inf would leave no differences.
    const float g = lane < count ? a.log_decay[at] : 0.0f;
    double total = static_cast<double>(g < -1.0e4f ? -1.0e4f : g) * kInverseLn2;
    const float strength = lane < count ? widen(a.beta[at]) : 0.0f;
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) {
      const double before = __shfl_up(total, step);
      if (lane >= step) total += before;
    }
    const float sum = static_cast<float>(total);
    const float rest = static_cast<float>(total - static_cast<double>(sum));
    wave_sync();  // the last head's values have been read
    mine.sum[lane] = sum;
    mine.rest[lane] = rest;
    mine.strength[lane] = strength;
    wave_sync();
    if ((wave & 1) == 0) {
      solve_head<kTrain>(s, mine, s.solve[wave >> 1], lane, block);
    } else {
      const double end = __shfl(total, 63);
      const float decay = __builtin_amdgcn_exp2f(sum);
      const float k_unit = lane < count ? s.k_unit[lane] : 0.0f;  // no rows past the end
      float* factors = reinterpret_cast<float*>(block);
      const float carry =
          __builtin_amdgcn_exp2f(static_cast<float>(end - total)) * k_unit;
      reinterpret_cast<f32x4*>(factors)[lane] =
          f32x4{decay * k_unit, strength, carry * strength,
                __builtin_amdgcn_exp2f(static_cast<float>(end))};
      factors[kCarry + lane] = carry;
      factors[kReadQuery + lane] = decay * s.q_unit[lane];
      factors[kSum + lane] = sum;
      factors[kSumRest + lane] = rest;
      read_out_head<kTrain>(s, mine, lane, block);
    }
  }
}

}  // namespace

int32_t launch_delta_prepare(void* stream, const RuleArgs& args, bf16_bits* outputs) {
  const dim3 grid(args.space.rows * args.space.key_heads), block(kThreads);
  return args.space.train
             ? launch(delta_prepare_kernel<true>, grid, block, stream, args, outputs)
             : launch(delta_prepare_kernel<false>, grid, block, stream, args, outputs);
}

}  // namespace gdn
