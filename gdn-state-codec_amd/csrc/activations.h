// Runs of 8 activations (bf16 or fp32) as fp32 registers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bf16_operands.h"

namespace gdn {

typedef uint16_t bf16_bits;

__device__ __forceinline__ float widen_low(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float widen_high(uint32_t pair) {
  return __uint_as_float(pair & 0xFFFF0000u);
}
__device__ __forceinline__ float widen(bf16_bits x) {
  return __uint_as_float(static_cast<uint32_t>(x) << 16);
}

// bf16 pair of two fp32 values, rounded to nearest even (NaN stays NaN).
__device__ __forceinline__ uint32_t bf16_pair(float low, float high) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){low, high}, bf16x2_t));
}

__device__ __forceinline__ void widen8(const uint4& w, float (&x)[8]) {
  x[0] = widen_low(w.x), x[1] = widen_high(w.x), x[2] = widen_low(w.y), x[3] = widen_high(w.y);
  x[4] = widen_low(w.z), x[5] = widen_high(w.z), x[6] = widen_low(w.w), x[7] = widen_high(w.w);
}

__device__ __forceinline__ uint4 narrow8(const float (&x)[8]) {
  return make_uint4(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4], x[5]),
                    bf16_pair(x[6], x[7]));
}

__device__ __forceinline__ void load8(const bf16_bits* p, float (&x)[8]) {
  widen8(*reinterpret_cast<const uint4*>(p), x);
}
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0];
  const float4 b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

__device__ __forceinline__ void store8(bf16_bits* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = narrow8(x);
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

}  // namespace gdn
