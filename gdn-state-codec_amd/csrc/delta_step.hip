// One token of the gated delta rule for every request of a batch, on a pool of
// dense [value][key] states.
//
// A row v of a head's state is independent of the others once k and q are known:
//   p = exp(g) (S_v . k),  u = b (v_v - p),  o_v = exp(g) (S_v . q) + u (k . q),
//   S_v <- exp(g) S_v + u k,
// so both products are taken on the old row in one pass, and the row is read
// once and written once: 128 KiB a head (fp32), which is what bounds the kernel
// (HBM; 5 fp32 operations a cell).
//
// 16 lanes hold a row, 8 keys each, so its two sums take four DPP exchanges and
// end in every lane that needs them: no LDS and no barrier, every wavefront on
// its own.  An fp32 row's lane holds keys 4l..4l+3 and 64+4l..64+4l+3 (each load
// instruction then covers whole 256-byte runs), a bf16 row's lane keys 8l..8l+7.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "activations.h"
#include "delta_chunk.h"
#include "gdn_state_codec_layer.h"
#include "lane_exchange.h"
#include "launch.h"
#include "stream_memory.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;
// Rows a wavefront.  One request's 32 heads (fp32) then take 3.5 us, 8 requests' 6.7 and
// 256 requests' 183 (1.07 GB, 5.9 TB/s); with 16 rows 4.0, 6.7 and 188, with 32 rows 5.2,
// 7.4 and 194.  Only between, at 16 requests, are 16 rows faster (10.7 and 12.8 us).
// From a bf16 pool 256 requests take 100 us (0.54 GB, 5.4 TB/s).
constexpr int kRows = 8;

struct StepArgs {
  const bf16_bits* queries;
  const bf16_bits* keys;
  const bf16_bits* values;
  const float* log_decay;
  const bf16_bits* beta;
  void* pool;
  const int32_t* slot_ids;
  bf16_bits* outputs;
  uint64_t query_stride, key_stride, value_stride;
  uint32_t batch, slots, value_heads, group;
  float scale;
  uint32_t normalize;
};

__device__ __forceinline__ float row_sum(float x) {  // over the 16 lanes of a row
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

template <typename Pool>
struct RowCells;

template <>
struct RowCells<float> {
  float4 low, high;
  __device__ __forceinline__ void load(const float* row, int l) {
    low = stream_load(reinterpret_cast<const float4*>(row + 4 * l));
    high = stream_load(reinterpret_cast<const float4*>(row + 64 + 4 * l));
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = low.x, x[1] = low.y, x[2] = low.z, x[3] = low.w;
    x[4] = high.x, x[5] = high.y, x[6] = high.z, x[7] = high.w;
  }
  static __device__ __forceinline__ void store(float* row, int l, const float (&x)[8]) {
    stream_store(reinterpret_cast<float4*>(row + 4 * l), make_float4(x[0], x[1], x[2], x[3]));
    stream_store(reinterpret_cast<float4*>(row + 64 + 4 * l),
                 make_float4(x[4], x[5], x[6], x[7]));
  }
  // The same keys of a bf16 vector.
  static __device__ __forceinline__ void vector(const bf16_bits* p, int l, float (&x)[8]) {
    const uint2 a = *reinterpret_cast<const uint2*>(p + 4 * l);
    const uint2 b = *reinterpret_cast<const uint2*>(p + 64 + 4 * l);
    widen8(make_uint4(a.x, a.y, b.x, b.y), x);
  }
};

template <>
struct RowCells<bf16_bits> {
  uint4 cells;
  __device__ __forceinline__ void load(const bf16_bits* row, int l) {
    cells = stream_load(reinterpret_cast<const uint4*>(row + 8 * l));
  }
  __device__ __forceinline__ void get(float (&x)[8]) const { widen8(cells, x); }
  static __device__ __forceinline__ void store(bf16_bits* row, int l, const float (&x)[8]) {
    const uint4 w = narrow8(x);  // the pool's own type: one rounding a token
    const u32x4_t v = {w.x, w.y, w.z, w.w};
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t*>(row + 8 * l));
  }
  static __device__ __forceinline__ void vector(const bf16_bits* p, int l, float (&x)[8]) {
    load8(p + 8 * l, x);
  }
};

// A wavefront takes kRows rows of one head, all asked for before the first is used.
template <typename Pool>
__global__ __launch_bounds__(kThreads) void delta_step_kernel(StepArgs a) {
  constexpr int kPasses = kRows / 4;
  constexpr int kWavesPerHead = kDim / kRows;
  const int lane = threadIdx.x & 63;
  const int l = lane & 15;
  const uint64_t wave = static_cast<uint64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
  const uint64_t tile = wave / kWavesPerHead;
  const uint32_t n = static_cast<uint32_t>(tile / a.value_heads);
  const uint32_t h = static_cast<uint32_t>(tile % a.value_heads);
  if (n >= a.batch) return;
  const int32_t slot = a.slot_ids[n];
  if (slot < 0 || static_cast<uint32_t>(slot) >= a.slots) return;
  const int first = static_cast<int>(wave % kWavesPerHead) * kRows + (lane >> 4);
  Pool* const state = static_cast<Pool*>(a.pool) +
                      (static_cast<uint64_t>(slot) * a.value_heads + h) * kTile +
                      first * kDim;
  RowCells<Pool> rows[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) rows[i].load(state + 4 * i * kDim, l);

  float q[8], k[8];
  RowCells<Pool>::vector(a.queries + n * a.query_stride + h / a.group * kDim, l, q);
  RowCells<Pool>::vector(a.keys + n * a.key_stride + h / a.group * kDim, l, k);
  float q_factor = a.scale, k_factor = 1.0f;
  if (a.normalize) {
    q_factor *= 1.0f / sqrtf(row_sum(dot8(q, q)) + kUnitEps);
    k_factor = 1.0f / sqrtf(row_sum(dot8(k, k)) + kUnitEps);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] *= q_factor;
    k[i] *= k_factor;
  }
  const float kq = row_sum(dot8(k, q));
  const uint64_t head = static_cast<uint64_t>(n) * a.value_heads + h;
  const float decay = expf(a.log_decay[head]);
  const float strength = widen(a.beta[head]);
  const bf16_bits* const values = a.values + n * a.value_stride + h * kDim + first;
  bf16_bits* const out = a.outputs + head * kDim + first;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    float s[8];
    rows[i].get(s);
    const float seen = decay * row_sum(dot8(s, k));
    const float read = decay * row_sum(dot8(s, q));
    const float u = strength * (widen(values[4 * i]) - seen);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = fmaf(u, k[j], decay * s[j]);
    RowCells<Pool>::store(state + 4 * i * kDim, l, s);
    if (l == 0) out[4 * i] = static_cast<bf16_bits>(bf16_pair(fmaf(u, kq, read), 0.0f));
  }
}

template <typename Pool>
int32_t launch_step(void* stream, const StepArgs& args) {
  const uint64_t blocks = static_cast<uint64_t>(args.batch) * args.value_heads *
                          (kDim / kRows) / (kThreads / 64);
  if (blocks > kMaxGrid) return kStatusInvalidArgument;
  return launch(delta_step_kernel<Pool>, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads),
                stream, args);
}

}  // namespace
}  // namespace gdn

extern "C" int32_t statecentric_gdn_state_codec_gated_delta_step_launch_v1(
    void* stream, const uint16_t* queries, const uint16_t* keys, const uint16_t* values,
    const float* log_decay, const uint16_t* beta, void* pool, const int32_t* slot_ids,
    uint16_t* outputs, uint32_t batch, uint32_t slots, uint32_t value_heads, uint32_t key_heads,
    uint64_t query_stride, uint64_t key_stride, uint64_t value_stride, uint32_t pool_dtype,
    float scale, uint32_t normalize) {
  if (!queries || !keys || !values || !log_decay || !beta || !pool || !slot_ids || !outputs ||
      batch == 0 || slots == 0 || key_heads == 0 || value_heads == 0 ||
      value_heads % key_heads != 0 || slots > 0x7FFFFFFFu || pool_dtype > gdn::kDtypeBF16 ||
      normalize > 1 || query_stride % 8 != 0 || key_stride % 8 != 0 || value_stride % 8 != 0 ||
      !gdn::element_aligned(log_decay, beta) ||
      !gdn::aligned16(queries, keys, values, pool, slot_ids, outputs)) {
    return gdn::kStatusInvalidArgument;
  }
  const gdn::StepArgs args{queries, keys, values, log_decay, beta, pool, slot_ids, outputs,
                           query_stride, key_stride, value_stride, batch, slots, value_heads,
                           value_heads / key_heads, scale, normalize};
  return pool_dtype == gdn::kDtypeF32 ? gdn::launch_step<float>(stream, args)
                                      : gdn::launch_step<gdn::bf16_bits>(stream, args);
}
