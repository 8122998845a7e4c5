// The norms around a gated-delta-net block, and their gradients.
//
// Before it, with the residual stream's update fused in (rows of `width`):
//   s = residual + scale x,   y = s r w,   r = 1 / sqrt(mean(s^2) + eps).
// After it, with the block's gate (rows of 128, one per head):
//   y = x r w z sigmoid(z).
// With n = s r (or x r) the normalized row and d the output's gradient,
//   d_n = d w (times z sigmoid(z)),   d_s = r (d_n - n mean(d_n n)),
//   d_w = sum over rows of d n (times z sigmoid(z)),
//   d_z = d n w sigmoid(z) (1 + z (1 - sigmoid(z))).
//
// Every kernel reads each input and writes each output once, which is what
// bounds it (HBM); a row stays in registers between its sum and its outputs.
// 8192 x 32 rows of 128 (bf16): forward 31 us (201 MB), backward 58 (335 MB, 5.8 TB/s)
// and 4 for the sum of its partials.  8192 rows of 4096 (bf16, fp32 stream): forward 72
// us (403 MB, 5.6 TB/s), backward 109 (537 MB, 4.9 TB/s) and 7.  256 rows of either:
// 3.2 us, a launch.
// Sums are fp32; each output is rounded once, to its own type.  The new residual
// stream is rounded before the norm is taken, so that y is the norm of what the
// next layer reads and the backward pass needs only the stored stream.
//
// d_w is a sum over all rows: each workgroup keeps its rows' part in registers,
// writes it to its own row of `partials`, and a second launch adds those rows in
// a fixed order (no atomics, so a call's result does not change from run to run).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "activations.h"
#include "gdn_state_codec_layer.h"
#include "lane_exchange.h"
#include "launch.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxWidth = 16384;

// sigmoid of a T on the transcendental unit (exp2 and reciprocal, about an ulp each).  The
// exponent's rounding puts up to |z| 2^-24 on the exponential: nothing beside a bf16
// value's own, but 65 x 2^-24 of an fp32 output at z = -80.  For fp32 what the product (and
// log2 e) left out is therefore put back as a factor: 6 x 2^-24 at any z.  The bounds, which
// only infinities and NaN reach, leave those what the exponential makes of them.
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  constexpr float kLog2E = 1.44269502162933349609375f, kLog2ERest = 1.92596303e-8f;
  constexpr float kLn2 = 0.693147180559945309f;
  const float t = -kLog2E * z;
  float power = __builtin_amdgcn_exp2f(t);
  if constexpr (sizeof(T) == sizeof(float)) {
    const float rest = fmaf(-kLog2ERest, z, fmaf(-kLog2E, z, -t));
    power *= fmaf(fminf(fmaxf(rest, -1.0e-4f), 1.0e-4f), kLn2, 1.0f);
  }
  return __builtin_amdgcn_rcpf(1.0f + power);
}

__device__ __forceinline__ float sum16(float x) {  // over the 16 lanes of a DPP row
  x = add_partner<1>(x);
  x = add_partner<2>(x);
  x = add_partner<4>(x);
  return add_partner<8>(x);
}

__device__ __forceinline__ float dot8(const float (&a)[8], const float (&b)[8]) {
  float x = a[0] * b[0], y = a[1] * b[1];
#pragma unroll
  for (int i = 2; i < 8; i += 2) {
    x = fmaf(a[i], b[i], x);
    y = fmaf(a[i + 1], b[i + 1], y);
  }
  return x + y;
}

// ---- the gated norm: 16 lanes a row, 8 columns a lane, 4 rows a wavefront ----

constexpr int kGatedRows = kThreads / 16;  // rows of a workgroup's pass

template <typename T>
__global__ __launch_bounds__(kThreads) void gated_norm_kernel(
    const T* __restrict__ x, const T* __restrict__ gate, const float* __restrict__ weight,
    T* __restrict__ out, uint64_t rows, float eps) {
  const int l = threadIdx.x & 15;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kGatedRows + (threadIdx.x >> 4);
  if (row >= rows) return;  // the same for a row's 16 lanes
  float v[8], z[8], w[8];
  load8(x + row * kDim + 8 * l, v);
  load8(gate + row * kDim + 8 * l, z);
  load8(weight + 8 * l, w);
  const float r = 1.0f / sqrtf(sum16(dot8(v, v)) * (1.0f / kDim) + eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w[i] * (z[i] * sigmoid<T>(z[i]));
  store8(out + row * kDim + 8 * l, v);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void gated_norm_backward_kernel(
    const T* __restrict__ x, const T* __restrict__ gate, const float* __restrict__ weight,
    const T* __restrict__ d_out, T* __restrict__ d_x, T* __restrict__ d_gate,
    float* __restrict__ partials, uint64_t rows, float eps) {
  __shared__ float parts[kGatedRows][kDim];
  const int l = threadIdx.x & 15;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kGatedRows;
  float w[8], d_w[8] = {};
  load8(weight + 8 * l, w);
  for (uint64_t row = static_cast<uint64_t>(blockIdx.x) * kGatedRows + (threadIdx.x >> 4);
       row < rows; row += step) {
    float v[8], z[8], d[8];
    load8(x + row * kDim + 8 * l, v);
    load8(gate + row * kDim + 8 * l, z);
    load8(d_out + row * kDim + 8 * l, d);
    const float r = 1.0f / sqrtf(sum16(dot8(v, v)) * (1.0f / kDim) + eps);
    float d_n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = sigmoid<T>(z[i]);
      v[i] *= r;  // the normalized row
      const float through = z[i] * s;
      const float dn = d[i] * v[i];
      d_w[i] = fmaf(dn, through, d_w[i]);
      d_n[i] = d[i] * w[i] * through;
      z[i] = dn * w[i] * (s * fmaf(z[i], 1.0f - s, 1.0f));  // d_gate
    }
    const float c = sum16(dot8(d_n, v)) * (1.0f / kDim);
#pragma unroll
    for (int i = 0; i < 8; ++i) d_n[i] = r * fmaf(-c, v[i], d_n[i]);
    store8(d_x + row * kDim + 8 * l, d_n);
    store8(d_gate + row * kDim + 8 * l, z);
  }
  store8(&parts[threadIdx.x >> 4][8 * l], d_w);
  __syncthreads();
  if (threadIdx.x < kDim) {
    float sum = parts[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < kGatedRows; ++i) sum += parts[i][threadIdx.x];
    partials[static_cast<uint64_t>(blockIdx.x) * kDim + threadIdx.x] = sum;
  }
}

// d_w[column] = sum over `count` partials, 8 columns a workgroup: 128 threads a column
// add every 128th row, four of them asked for at a time, and one wavefront adds their
// sums in a fixed order.
constexpr int kSumThreads = 1024;
constexpr int kSumGroups = kSumThreads / 8;

__global__ __launch_bounds__(kSumThreads) void weight_sum_kernel(
    const float* __restrict__ partials, float* __restrict__ d_weight, uint32_t count,
    uint32_t width) {
  __shared__ float parts[kSumGroups][9];
  const int column = threadIdx.x & 7;
  const uint32_t group = threadIdx.x >> 3;
  const float* p = partials + 8 * static_cast<uint64_t>(blockIdx.x) + column;
  float sum = 0.0f;
  for (uint32_t i = group; i < count; i += 4 * kSumGroups) {
    float x[4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      x[u] = p[static_cast<uint64_t>(min(i + u * kSumGroups, count - 1)) * width];
    }
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) sum += i + u * kSumGroups < count ? x[u] : 0.0f;
  }
  parts[group][column] = sum;
  __syncthreads();
  if (threadIdx.x < 64) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < kSumGroups / 8; ++i) total += parts[kSumGroups / 8 * group + i][column];
    total += __shfl_xor(total, 8);
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);
    if (group == 0) d_weight[8 * blockIdx.x + column] = total;
  }
}

// ---- the residual norm: kSpan threads a row, kRuns runs of 8 columns each ----
// A wavefront takes a row of up to 1024 columns (no barrier); a workgroup takes a
// wider one, at most 8 runs (64 columns) a thread.

template <int kSpan>
__device__ __forceinline__ float row_total(float x, float (&waves)[2][4], int turn) {
  x = wave_sum_valu(x);
  if constexpr (kSpan == 256) {
    if ((threadIdx.x & 63) == 0) waves[turn][threadIdx.x >> 6] = x;
    __syncthreads();
    x = (waves[turn][0] + waves[turn][1]) + (waves[turn][2] + waves[turn][3]);
  }
  return x;
}

template <typename T>
__device__ __forceinline__ void round8(float (&x)[8]);
template <>
__device__ __forceinline__ void round8<float>(float (&)[8]) {}
template <>
__device__ __forceinline__ void round8<bf16_bits>(float (&x)[8]) {
  widen8(narrow8(x), x);
}

template <typename T, typename S, int kSpan, int kRuns>
__global__ __launch_bounds__(kThreads) void residual_norm_kernel(
    const T* __restrict__ x, const S* residual, const float* __restrict__ weight,
    T* __restrict__ out, S* sum, uint64_t rows, uint32_t width, float scale, float eps) {
  __shared__ float waves[2][4];
  const uint32_t t = threadIdx.x % kSpan;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (kThreads / kSpan) +
                       threadIdx.x / kSpan;
  const bool live = row < rows;  // uniform over a wavefront (kSpan 64) or workgroup
  const uint64_t base = row * width;
  float s[kRuns][8];
  float squares = 0.0f;
#pragma unroll
  for (int j = 0; j < kRuns; ++j) {
    const uint32_t at = 8 * (j * kSpan + t);
    if (live && at < width) {
      float v[8];
      load8(x + base + at, v);
      load8(residual + base + at, s[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[j][i] = fmaf(scale, v[i], s[j][i]);
      round8<S>(s[j]);
      store8(sum + base + at, s[j]);
      squares += dot8(s[j], s[j]);
    }
  }
  const float r = 1.0f / sqrtf(row_total<kSpan>(squares, waves, 0) / static_cast<float>(width) +
                               eps);
#pragma unroll
  for (int j = 0; j < kRuns; ++j) {
    const uint32_t at = 8 * (j * kSpan + t);
    if (live && at < width) {
      float w[8];
      load8(weight + at, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[j][i] = s[j][i] * r * w[i];
      store8(out + base + at, s[j]);
    }
  }
}

template <typename T, typename S, int kSpan, int kRuns>
__global__ __launch_bounds__(kThreads) void residual_norm_backward_kernel(
    const S* __restrict__ sum, const float* __restrict__ weight, const T* __restrict__ d_out,
    const S* __restrict__ d_sum, T* __restrict__ d_x, S* __restrict__ d_residual,
    float* __restrict__ partials, uint64_t rows, uint32_t width, float scale, float eps) {
  constexpr int kRows = kThreads / kSpan;
  __shared__ float waves[2][4];
  __shared__ float parts[kRows == 1 ? 1 : kRows * kSpan * kRuns * 8];
  const uint32_t t = threadIdx.x % kSpan;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kRows;
  const float by_width = 1.0f / static_cast<float>(width);
  float d_w[kRuns][8] = {};
  for (uint64_t row = static_cast<uint64_t>(blockIdx.x) * kRows + threadIdx.x / kSpan; row < rows;
       row += step) {  // uniform over a wavefront (kSpan 64) or workgroup
    const uint64_t base = row * width;
    float s[kRuns][8], d[kRuns][8];
    float squares = 0.0f, along = 0.0f;
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
      const uint32_t at = 8 * (j * kSpan + t);
      if (at < width) {
        float w[8];
        load8(sum + base + at, s[j]);
        load8(d_out + base + at, d[j]);
        load8(weight + at, w);
        squares += dot8(s[j], s[j]);
        float dw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[i] = d[j][i] * w[i];
        along += dot8(dw, s[j]);
      }
    }
    const float r = 1.0f / sqrtf(row_total<kSpan>(squares, waves, 0) * by_width + eps);
    const float c = row_total<kSpan>(along, waves, 1) * r * by_width;  // mean(d_n n)
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
      const uint32_t at = 8 * (j * kSpan + t);
      if (at < width) {
        float w[8], more[8] = {};
        load8(weight + at, w);
        if (d_sum != nullptr) load8(d_sum + base + at, more);
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float n = s[j][i] * r;
          d_w[j][i] = fmaf(d[j][i], n, d_w[j][i]);
          g[i] = fmaf(r, fmaf(-c, n, d[j][i] * w[i]), more[i]);
        }
        store8(d_residual + base + at, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= scale;
        store8(d_x + base + at, g);
      }
    }
    // With kSpan 256 the second sum's barrier lies between every thread's read of
    // waves[0] and the next row's write of it, and the next row's first barrier
    // between the reads of waves[1] and its next write.
  }
  float* const mine = partials + static_cast<uint64_t>(blockIdx.x) * width;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
      const uint32_t at = 8 * (j * kSpan + t);
      if (at < width) store8(mine + at, d_w[j]);
    }
  } else {  // join the wavefronts' rows
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
      store8(parts + (threadIdx.x / kSpan) * (kSpan * kRuns * 8) + 8 * (j * kSpan + t), d_w[j]);
    }
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < width; at += kThreads) {
      float total = parts[at];
#pragma unroll
      for (int i = 1; i < kRows; ++i) total += parts[i * (kSpan * kRuns * 8) + at];
      mine[at] = total;
    }
  }
}

// Workgroups of a backward pass, and so rows of its partials: enough to fill the
// chip several times over, few enough that the partials stay a small share of
// the traffic (2% at 8192 rows of 4096).
uint32_t most_partials(uint64_t rows, uint32_t width) {
  const uint64_t passes = (rows + 3) / 4;
  const uint32_t most = width <= 512 ? 1024 : 512;
  return passes < most ? static_cast<uint32_t>(passes) : most;
}

int32_t add_partials(void* stream, const float* partials, float* d_weight, uint32_t count,
                     uint32_t width) {
  return launch(weight_sum_kernel, dim3(width / 8), dim3(kSumThreads), stream, partials, d_weight,
                count, width);
}

template <typename T>
int32_t gated_backward(void* stream, const void* x, const void* gate, const float* weight,
                       const void* d_out, void* d_x, void* d_gate, float* d_weight,
                       float* partials, uint64_t rows, float eps) {
  const uint64_t passes = (rows + kGatedRows - 1) / kGatedRows;
  const uint32_t most = most_partials(rows, kDim);
  const uint32_t blocks = passes < most ? static_cast<uint32_t>(passes) : most;
  const int32_t status = launch(gated_norm_backward_kernel<T>, dim3(blocks), dim3(kThreads),
                                stream, static_cast<const T*>(x), static_cast<const T*>(gate),
                                weight, static_cast<const T*>(d_out), static_cast<T*>(d_x),
                                static_cast<T*>(d_gate), partials, rows, eps);
  return status != kStatusOk ? status : add_partials(stream, partials, d_weight, blocks, kDim);
}

struct ResidualArgs {
  const void* x;
  const void* residual;
  const float* weight;
  void* out;
  void* sum;
  const void* d_out;
  const void* d_sum;
  void* d_x;
  void* d_residual;
  float* d_weight;
  float* partials;
  uint64_t rows;
  uint32_t width;
  float scale, eps;
};

template <typename T, typename S, int kSpan, int kRuns>
int32_t residual_launch(void* stream, const ResidualArgs& a, bool backward) {
  constexpr int kRows = kThreads / kSpan;
  const uint64_t passes = (a.rows + kRows - 1) / kRows;
  if (!backward) {
    if (passes > kMaxGrid) return kStatusInvalidArgument;
    return launch(residual_norm_kernel<T, S, kSpan, kRuns>, dim3(static_cast<uint32_t>(passes)),
                  dim3(kThreads), stream, static_cast<const T*>(a.x),
                  static_cast<const S*>(a.residual), a.weight, static_cast<T*>(a.out),
                  static_cast<S*>(a.sum), a.rows, a.width, a.scale, a.eps);
  }
  const uint32_t most = most_partials(a.rows, a.width);
  const uint32_t blocks = passes < most ? static_cast<uint32_t>(passes) : most;
  const int32_t status = launch(
      residual_norm_backward_kernel<T, S, kSpan, kRuns>, dim3(blocks), dim3(kThreads), stream,
      static_cast<const S*>(a.sum), a.weight, static_cast<const T*>(a.d_out),
      static_cast<const S*>(a.d_sum), static_cast<T*>(a.d_x), static_cast<S*>(a.d_residual),
      a.partials, a.rows, a.width, a.scale, a.eps);
  return status != kStatusOk ? status
                             : add_partials(stream, a.partials, a.d_weight, blocks, a.width);
}

template <typename T, typename S>
int32_t residual_by_width(void* stream, const ResidualArgs& a, bool backward) {
  if (a.width <= 512) return residual_launch<T, S, 64, 1>(stream, a, backward);
  if (a.width <= 1024) return residual_launch<T, S, 64, 2>(stream, a, backward);
  if (a.width <= 2048) return residual_launch<T, S, 256, 1>(stream, a, backward);
  if (a.width <= 4096) return residual_launch<T, S, 256, 2>(stream, a, backward);
  if (a.width <= 8192) return residual_launch<T, S, 256, 4>(stream, a, backward);
  return residual_launch<T, S, 256, 8>(stream, a, backward);
}

int32_t residual_by_type(void* stream, const ResidualArgs& a, uint32_t dtype,
                         uint32_t stream_dtype, bool backward) {
  if (dtype == kDtypeF32) {
    return stream_dtype == kDtypeF32 ? residual_by_width<float, float>(stream, a, backward)
                                     : residual_by_width<float, bf16_bits>(stream, a, backward);
  }
  return stream_dtype == kDtypeF32 ? residual_by_width<bf16_bits, float>(stream, a, backward)
                                   : residual_by_width<bf16_bits, bf16_bits>(stream, a, backward);
}

// Rows whose last element's index fits 63 bits, and a width the kernels divide.
bool residual_shape_ok(uint64_t rows, uint32_t width, uint32_t dtype, uint32_t stream_dtype) {
  return rows > 0 && rows <= 1ull << 40 && width > 0 && width <= kMaxWidth && width % 8 == 0 &&
         dtype <= kDtypeBF16 && stream_dtype <= kDtypeBF16;
}

}  // namespace
}  // namespace gdn

extern "C" uint32_t statecentric_gdn_state_codec_norm_partials_v1(uint64_t rows,
                                                                  uint32_t width) {
  return gdn::most_partials(rows, width);
}

extern "C" int32_t statecentric_gdn_state_codec_gated_norm_launch_v1(
    void* stream, const void* x, const void* gate, const float* weight, void* out, uint64_t rows,
    uint32_t dtype, float eps) {
  const uint64_t blocks = rows / gdn::kGatedRows + (rows % gdn::kGatedRows != 0 ? 1 : 0);
  if (!x || !gate || !weight || !out || rows == 0 || blocks > gdn::kMaxGrid ||
      dtype > gdn::kDtypeBF16 || !gdn::aligned16(x, gate, weight, out)) {
    return gdn::kStatusInvalidArgument;
  }
  const dim3 grid(static_cast<uint32_t>(blocks)), block(gdn::kThreads);
  if (dtype == gdn::kDtypeF32) {
    return gdn::launch(gdn::gated_norm_kernel<float>, grid, block, stream,
                       static_cast<const float*>(x), static_cast<const float*>(gate), weight,
                       static_cast<float*>(out), rows, eps);
  }
  return gdn::launch(gdn::gated_norm_kernel<gdn::bf16_bits>, grid, block, stream,
                     static_cast<const gdn::bf16_bits*>(x),
                     static_cast<const gdn::bf16_bits*>(gate), weight,
                     static_cast<gdn::bf16_bits*>(out), rows, eps);
}

extern "C" int32_t statecentric_gdn_state_codec_gated_norm_backward_launch_v1(
    void* stream, const void* x, const void* gate, const float* weight, const void* d_out,
    void* d_x, void* d_gate, float* d_weight, float* partials, uint64_t rows, uint32_t dtype,
    float eps) {
  if (!x || !gate || !weight || !d_out || !d_x || !d_gate || !d_weight || !partials ||
      rows == 0 || rows > 1ull << 40 || dtype > gdn::kDtypeBF16 ||
      !gdn::aligned16(x, gate, weight, d_out, d_x, d_gate, d_weight, partials)) {
    return gdn::kStatusInvalidArgument;
  }
  return dtype == gdn::kDtypeF32
             ? gdn::gated_backward<float>(stream, x, gate, weight, d_out, d_x, d_gate, d_weight,
                                          partials, rows, eps)
             : gdn::gated_backward<gdn::bf16_bits>(stream, x, gate, weight, d_out, d_x, d_gate,
                                                   d_weight, partials, rows, eps);
}

extern "C" int32_t statecentric_gdn_state_codec_residual_norm_launch_v1(
    void* stream, const void* x, const void* residual, const float* weight, void* out, void* sum,
    uint64_t rows, uint32_t width, uint32_t dtype, uint32_t stream_dtype, float scale, float eps) {
  if (!x || !residual || !weight || !out || !sum ||
      !gdn::residual_shape_ok(rows, width, dtype, stream_dtype) ||
      !gdn::aligned16(x, residual, weight, out, sum)) {
    return gdn::kStatusInvalidArgument;
  }
  gdn::ResidualArgs a{};
  a.x = x, a.residual = residual, a.weight = weight, a.out = out, a.sum = sum;
  a.rows = rows, a.width = width, a.scale = scale, a.eps = eps;
  return gdn::residual_by_type(stream, a, dtype, stream_dtype, false);
}

extern "C" int32_t statecentric_gdn_state_codec_residual_norm_backward_launch_v1(
    void* stream, const void* sum, const float* weight, const void* d_out, const void* d_sum,
    void* d_x, void* d_residual, float* d_weight, float* partials, uint64_t rows, uint32_t width,
    uint32_t dtype, uint32_t stream_dtype, float scale, float eps) {
  if (!sum || !weight || !d_out || !d_x || !d_residual || !d_weight || !partials ||
      !gdn::residual_shape_ok(rows, width, dtype, stream_dtype) ||
      !gdn::aligned16(sum, weight, d_out, d_sum, d_x, d_residual, d_weight, partials)) {
    return gdn::kStatusInvalidArgument;
  }
  gdn::ResidualArgs a{};
  a.sum = const_cast<void*>(sum), a.weight = weight, a.d_out = d_out, a.d_sum = d_sum;
  a.d_x = d_x, a.d_residual = d_residual, a.d_weight = d_weight, a.partials = partials;
  a.rows = rows, a.width = width, a.scale = scale, a.eps = eps;
  return gdn::residual_by_type(stream, a, dtype, stream_dtype, true);
}
