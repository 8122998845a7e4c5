// The state-independent half of the gated delta rule's chunked form, for every
// chunk and key head at once: the operands K, Q and their transposes, the norms,
// and for each value head of the group the factors, N and P b (and for training
// N^T and P^T); formulas and layouts in delta_chunk.h.
//
// One workgroup per chunk row and key head.  K K^T and Q K^T are formed once per
// key head on the matrix cores (exact bf16 products).  N comes from forward
// substitution, one column a lane: lane j keeps N_1j..N_63j in registers, and the
// rows of A b come from LDS as broadcasts (every lane reads the same 16 bytes).
// That is 2016 fp32 fmas a wavefront, the kernel's bound together with their
// broadcasts; substitution is stable for any keys, which powers of A are not.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "delta_chunk.h"
#include "lane_exchange.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr int kPitch = 136;  // bf16 a staged row: 128 and 16 bytes against bank conflicts
constexpr int kWide = 68;    // fp32 a row of a 64 x 64 matrix

struct Staged {
  union {
    struct {
      uint16_t k[kChunk][kPitch];
      uint16_t q[kChunk][kPitch];
    };
    float solve[2][kChunk][kWide];  // A b, then N, of two value heads
  };
  float kk[kChunk][kWide];
  float qk[kChunk][kWide];
  double sum[2][kChunk];    // G
  float strength[2][kChunk];
  float k_unit[kChunk];     // 1 / |k|
  float q_unit[kChunk];     // scale / |q|
  float q_norm[kChunk];     // 1 / |q|
};

// LDS written by other lanes of the same wavefront is read after this.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

__device__ __forceinline__ int place(int step, int g, int i) {  // of a contraction
  return 32 * step + (i < 4 ? 4 * g + i : 12 + 4 * g + i);
}

__device__ __forceinline__ void store_parts(char* tiles, int tile, int lane,
                                            const uint4 (&part)[3], int parts) {
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    if (p < parts) {
      reinterpret_cast<uint4*>(tiles + (p * kTriangle + tile) * kTileBytes)[lane] = part[p];
    }
  }
}

// Forward substitution of one value head by one wavefront, and N's operands.
template <bool kTrain>
__device__ __forceinline__ void solve_head(Staged& s, int slot, int lane, char* block) {
  float (&m)[kChunk][kWide] = s.solve[slot];
  const double mine = s.sum[slot][lane];
  const float k_mine = s.k_unit[lane], b_mine = s.strength[slot][lane];
  float n[kChunk];  // column `lane`
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const float decay = expf(static_cast<float>(s.sum[slot][i] - mine));
    const float a = i > lane ? decay * (s.k_unit[i] * k_mine * s.kk[i][lane]) : 0.0f;
    n[i] = -a;
    m[i][lane] = a * b_mine;
  }
  wave_sync();
#pragma unroll
  for (int i = 1; i < kChunk; ++i) {
    float sum[4] = {n[i], 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < i; j += 4) {
      const f32x4 row = load4(&m[i][j]);  // zero from the diagonal on
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (j + c < i) sum[c] = fmaf(-row[c], n[j + c], sum[c]);
      }
    }
    n[i] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }
  wave_sync();  // A b has been read
#pragma unroll
  for (int i = 0; i < kChunk; ++i) m[i][lane] = n[i];
  wave_sync();
  const int row = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      uint4 part[3];
      if (step < lower_steps(t)) {
        const float* p = &m[16 * t + row][32 * step + 4 * g];
        split3(load4(p), load4(p + 16), part);
        store_parts(block + kSolve, lower_tile(t, step), lane, part, kSolveParts);
      }
      if (kTrain && step >= upper_first(t)) {
        f32x4 x, y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = m[place(step, g, i)][16 * t + row];
          y[i] = m[place(step, g, i + 4)][16 * t + row];
        }
        split3(x, y, part);
        store_parts(block + kSolveBack, upper_tile(t, step), lane, part, kSolveParts);
      }
    }
  }
}

// P b of one value head (and P^T) by one wavefront.
template <bool kTrain>
__device__ __forceinline__ void read_out_head(const Staged& s, int slot, int lane, char* block) {
  const int row = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int at = 16 * t + row;
    const double mine = s.sum[slot][at];
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      f32x4 x[2];
      uint4 part[3];
      if (step < lower_steps(t)) {  // row i = at, columns j
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = place(step, g, i);
          const float decay = expf(static_cast<float>(mine - s.sum[slot][j]));
          x[i / 4][i % 4] = j <= at ? decay * (s.q_unit[at] * s.k_unit[j] * s.qk[at][j]) *
                                          s.strength[slot][j]
                                    : 0.0f;
        }
        // Two parts, rounded: 2^-16 of a weight whose sums become bf16 outputs.
        split2_pair(x[0][0], x[0][1], part[0].x, part[1].x);
        split2_pair(x[0][2], x[0][3], part[0].y, part[1].y);
        split2_pair(x[1][0], x[1][1], part[0].z, part[1].z);
        split2_pair(x[1][2], x[1][3], part[0].w, part[1].w);
        store_parts(block + kReadOut, lower_tile(t, step), lane, part, kReadParts);
      }
      if (kTrain && step >= upper_first(t)) {  // row j = at, columns i
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int token = place(step, g, i);
          const float decay = expf(static_cast<float>(s.sum[slot][token] - mine));
          x[i / 4][i % 4] =
              at <= token ? decay * (s.q_unit[token] * s.k_unit[at] * s.qk[token][at]) : 0.0f;
        }
        split3(x[0], x[1], part);
        store_parts(block + kReadBack, upper_tile(t, step), lane, part, kSolveParts);
      }
    }
  }
}

// The outputs of tokens of no request: zeros, for one key head's value heads.
__device__ __forceinline__ void clear_rest(const RuleArgs& a, uint32_t head,
                                           bf16_bits* outputs) {
  const uint32_t from = min(static_cast<uint32_t>(a.offsets[a.requests]), a.tokens);
  const uint32_t width = a.group * kDim;
  for (uint64_t i = threadIdx.x; i < static_cast<uint64_t>(a.tokens - from) * width;
       i += kThreads) {
    outputs[(from + i / width) * a.space.value_heads * kDim + head * width + i % width] = 0;
  }
}

template <bool kTrain>
__global__ __launch_bounds__(kThreads) void delta_prepare_kernel(RuleArgs a,
                                                                bf16_bits* outputs) {
  __shared__ Staged s;
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const uint32_t row = blockIdx.x / a.space.key_heads;
  const uint32_t head = blockIdx.x % a.space.key_heads;
  const int4 chunk = a.chunks[row];
  const int count = chunk_tokens(a, chunk);
  if (kTrain && row == 0) clear_rest(a, head, outputs);
  if (count == 0 || (!kTrain && chunk.w < 0)) return;  // past the last chunk, or padding
  const uint64_t first = chunk.y;

  {  // stage the rows, 32 columns a thread, zeros past the request's end
    const int token = t >> 2, part = t & 3;
    float kk = 0.0f, qq = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 k = make_uint4(0, 0, 0, 0), q = k;
      const int column = 32 * part + 8 * i;
      if (token < count) {
        k = *reinterpret_cast<const uint4*>(a.keys + (first + token) * a.key_stride +
                                            head * kDim + column);
        q = *reinterpret_cast<const uint4*>(a.queries + (first + token) * a.query_stride +
                                            head * kDim + column);
      }
      *reinterpret_cast<uint4*>(&s.k[token][column]) = k;
      *reinterpret_cast<uint4*>(&s.q[token][column]) = q;
      float x[8];
      widen8(k, x);
#pragma unroll
      for (int c = 0; c < 8; ++c) kk = fmaf(x[c], x[c], kk);
      widen8(q, x);
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
  {  // row tile `wave` of K K^T and Q K^T, up to the diagonal
    uint4 k[4], q[4];
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      k[step] = *reinterpret_cast<const uint4*>(&s.k[16 * wave + r][32 * step + 8 * g]);
      q[step] = *reinterpret_cast<const uint4*>(&s.q[16 * wave + r][32 * step + 8 * g]);
    }
    for (int c = 0; c <= wave; ++c) {
      f32x4 kk = {0.0f, 0.0f, 0.0f, 0.0f}, qk = kk;
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        const uint4 b = *reinterpret_cast<const uint4*>(&s.k[16 * c + r][32 * step + 8 * g]);
        kk = mfma(k[step], b, kk);
        qk = mfma(q[step], b, qk);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s.kk[16 * wave + 4 * g + i][16 * c + r] = kk[i];
        s.qk[16 * wave + 4 * g + i][16 * c + r] = qk[i];
      }
    }
    // Its rows as operands over the keys.
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const uint16_t* k_row = &s.k[16 * wave + r][32 * step + 4 * g];
      const uint16_t* q_row = &s.q[16 * wave + r][32 * step + 4 * g];
      const uint2 k0 = *reinterpret_cast<const uint2*>(k_row);
      const uint2 k1 = *reinterpret_cast<const uint2*>(k_row + 16);
      const uint2 q0 = *reinterpret_cast<const uint2*>(q_row);
      const uint2 q1 = *reinterpret_cast<const uint2*>(q_row + 16);
      const int tile = (4 * wave + step) * kTileBytes;
      reinterpret_cast<uint4*>(key_block + kKeyRows + tile)[lane] =
          make_uint4(k0.x, k0.y, k1.x, k1.y);
      reinterpret_cast<uint4*>(key_block + kQueryRows + tile)[lane] =
          make_uint4(q0.x, q0.y, q1.x, q1.y);
    }
    // Two row tiles of the transposes: rows = keys, over the tokens.
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int key = 32 * wave + 16 * c + r;
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        uint32_t kw[4], qw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int x = place(step, g, 2 * i), y = place(step, g, 2 * i + 1);
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

  // Value heads two at a time: wavefronts 0 and 1 solve, 2 and 3 form P b.
  for (uint32_t pair = 0; pair < a.group; pair += 2) {
    __syncthreads();  // K and Q (or the last pair's N and factors) have been read
    const int slot = wave & 1;
    const uint32_t member = pair + slot;
    const bool live = member < a.group;
    const uint32_t value_head = head * a.group + (live ? member : 0);
    char* const block = a.space.value_block(row, value_head);
    if (wave < 2 && live) {
      const uint64_t at = (first + lane) * a.space.value_heads + value_head;
      double sum = lane < count ? static_cast<double>(a.log_decay[at]) : 0.0;
      const float strength = lane < count ? widen(a.beta[at]) : 0.0f;
#pragma unroll
      for (int step = 1; step < 64; step <<= 1) {
        const double before = __shfl_up(sum, step);
        if (lane >= step) sum += before;
      }
      s.sum[slot][lane] = sum;
      s.strength[slot][lane] = strength;
      const double end = __shfl(sum, 63);
      const float decay = expf(static_cast<float>(sum));
      float* factors = reinterpret_cast<float*>(block);
      factors[kReadKey * kChunk + lane] = decay * s.k_unit[lane];
      factors[kReadQuery * kChunk + lane] = decay * s.q_unit[lane];
      factors[kStrength * kChunk + lane] = strength;
      factors[kWrite * kChunk + lane] =
          expf(static_cast<float>(end - sum)) * s.k_unit[lane];
      factors[kSum * kChunk + lane] = static_cast<float>(sum);
      factors[kSumRest * kChunk + lane] =
          static_cast<float>(sum - static_cast<double>(static_cast<float>(sum)));
      factors[kWhole * kChunk + lane] = expf(static_cast<float>(end));
    }
    __syncthreads();
    if (live) {
      if (wave < 2) solve_head<kTrain>(s, slot, lane, block);
      else read_out_head<kTrain>(s, slot, lane, block);
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
