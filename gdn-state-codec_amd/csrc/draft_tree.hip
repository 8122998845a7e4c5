// The gated delta rule over a tree of drafted tokens of each request, read from its
// cached state, and that state after an accepted path.
//
// With S0 the cached state of one value head ([value][key]), G_t the sum of the log
// decays from it down to node t, b_t the write strength, unit keys k and scaled unit
// queries q:
//   u_t = b_t (v_t - exp(G_t) S0 k_t - sum_(i above t) exp(G_t - G_i) (k_i . k_t) u_i)
//   o_t = exp(G_t) S0 q_t + sum_(i above t, and t) exp(G_t - G_i) (k_i . q_t) u_i
// and after the path down to node c
//   S = exp(G_c) S0 + sum_(i on the path) exp(G_c - G_i) u_i k_i^T.
//
// A workgroup takes one head of one request, a thread one row of its state; the products
// of the nodes' keys and queries are formed once, in LDS.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "delta_chunk.h"
#include "gdn_state_codec_layer.h"
#include "launch.h"

namespace gdn {
namespace {

constexpr int kMaxNodes = GDN_STATE_CODEC_MAX_NODES;

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

struct Shared {
  float k[kMaxNodes][kDim + 1], q[kMaxNodes][kDim + 1];
  float u[kMaxNodes][kDim];
  float kk[kMaxNodes][kMaxNodes], qk[kMaxNodes][kMaxNodes];
  float decay[kMaxNodes], strength[kMaxNodes];
  int parent[kMaxNodes];
};

__device__ __forceinline__ float cell(const float* p) { return *p; }
__device__ __forceinline__ float cell(const bf16_bits* p) { return widen(*p); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(bf16_bits* p, float x) {
  *p = static_cast<bf16_bits>(bf16_pair(x, 0.0f));
}

template <typename Pool, bool kCommit>
__global__ __launch_bounds__(kDim) void draft_kernel(DraftArgs a) {
  __shared__ Shared s;
  const int t = threadIdx.x;
  const uint32_t r = blockIdx.x / a.value_heads, h = blockIdx.x % a.value_heads;
  const int32_t slot = a.slot_ids[r];
  if (slot < 0 || static_cast<uint32_t>(slot) >= a.slots) return;
  const int64_t begin = max(a.offsets[r], 0);
  const int64_t end = min(static_cast<int64_t>(a.offsets[r + 1]), static_cast<int64_t>(a.tokens));
  const int nodes = static_cast<int>(min(end - begin, static_cast<int64_t>(a.max_nodes)));
  if (nodes <= 0) return;
  int last = nodes - 1;
  if (kCommit) {
    last = a.accepted[r];
    if (last < 0 || last >= nodes) return;
  }
  for (int i = 0; i < nodes; ++i) {
    const uint64_t row = begin + i;
    s.k[i][t] = widen(a.keys[row * a.key_stride + h / a.group * kDim + t]);
    if (!kCommit) s.q[i][t] = widen(a.queries[row * a.query_stride + h / a.group * kDim + t]);
  }
  if (t < nodes) {
    const uint64_t row = begin + t;
    const int p = a.parents[row];
    s.parent[t] = p < 0 || p >= t ? -1 : p;
    s.decay[t] = expf(a.log_decay[row * a.value_heads + h]);
    s.strength[t] = widen(a.beta[row * a.value_heads + h]);
  }
  __syncthreads();
  if (t < nodes) {
    float kk = kUnitEps, qq = kUnitEps;
    for (int j = 0; j < kDim; ++j) {
      kk = fmaf(s.k[t][j], s.k[t][j], kk);
      if (!kCommit) qq = fmaf(s.q[t][j], s.q[t][j], qq);
    }
    const float k_unit = a.normalize ? 1.0f / sqrtf(kk) : 1.0f;
    const float q_unit = a.normalize ? a.scale / sqrtf(qq) : a.scale;
    for (int j = 0; j < kDim; ++j) {
      s.k[t][j] *= k_unit;
      if (!kCommit) s.q[t][j] *= q_unit;
    }
  }
  __syncthreads();
  for (int pair = t; pair < nodes * nodes; pair += kDim) {
    const int i = pair / nodes, j = pair % nodes;
    if (j > i) continue;
    float kk = 0.0f, qk = 0.0f;
    for (int d = 0; d < kDim; ++d) {
      kk = fmaf(s.k[i][d], s.k[j][d], kk);
      if (!kCommit) qk = fmaf(s.q[i][d], s.k[j][d], qk);
    }
    s.kk[i][j] = kk;
    if (!kCommit) s.qk[i][j] = qk;
  }
  __syncthreads();
  Pool* const state = static_cast<Pool*>(a.pool) +
                      (static_cast<uint64_t>(slot) * a.value_heads + h) * kTile + t * kDim;
  uint64_t on_path = 0;
  if (kCommit) {
    for (int i = last; i >= 0; i = s.parent[i]) on_path |= 1ull << i;
  }
  for (int i = 0; i <= last; ++i) {
    if (kCommit && !(on_path >> i & 1)) continue;
    const uint64_t row = begin + i;
    float seen = 0.0f, read = 0.0f;
    for (int j = 0; j < kDim; ++j) {
      const float x = cell(state + j);
      seen = fmaf(x, s.k[i][j], seen);
      if (!kCommit) read = fmaf(x, s.q[i][j], read);
    }
    float decay = s.decay[i], seen_writes = 0.0f, read_writes = 0.0f;
    for (int j = s.parent[i]; j >= 0; j = s.parent[j]) {
      const float u = decay * s.u[j][t];
      seen_writes = fmaf(u, s.kk[i][j], seen_writes);
      if (!kCommit) read_writes = fmaf(u, s.qk[i][j], read_writes);
      decay *= s.decay[j];
    }
    const float v = widen(a.values[row * a.value_stride + h * kDim + t]);
    const float u = s.strength[i] * (v - fmaf(decay, seen, seen_writes));
    s.u[i][t] = u;  // read by this thread alone
    if (!kCommit) {
      put(a.outputs + (row * a.value_heads + h) * kDim + t,
          fmaf(u, s.qk[i][i], fmaf(decay, read, read_writes)));
    }
  }
  if (kCommit) {
    for (int j = 0; j < kDim; ++j) {
      float decay = 1.0f, x = 0.0f;
      for (int i = last; i >= 0; i = s.parent[i]) {
        x = fmaf(decay * s.u[i][t], s.k[i][j], x);
        decay *= s.decay[i];
      }
      put(state + j, fmaf(decay, cell(state + j), x));
    }
  }
}

template <bool kCommit>
int32_t launch_drafts(void* stream, const gdn_state_codec_drafts* d, const int32_t* accepted,
                      void* pool, uint32_t slots, uint32_t pool_dtype, uint16_t* outputs) {
  if (!d || !pool || slots == 0 || slots > 0x7FFFFFFFu || pool_dtype > kDtypeBF16 ||
      d->requests == 0 || d->requests > GDN_STATE_CODEC_MAX_REQUESTS ||
      d->tokens > 0x7FFFFFFFu || d->key_heads == 0 || d->value_heads == 0 ||
      d->value_heads % d->key_heads != 0 || d->max_nodes == 0 || d->max_nodes > kMaxNodes ||
      d->normalize > 1 || d->query_stride % 8 != 0 || d->key_stride % 8 != 0 ||
      d->value_stride % 8 != 0 || !d->offsets || !d->slot_ids ||
      !token_rows(d->tokens, d->keys, d->values, d->log_decay, d->beta, d->parents) ||
      (kCommit ? !accepted || d->queries != nullptr
               : !token_rows(d->tokens, d->queries, outputs)) ||
      reinterpret_cast<uintptr_t>(d->parents) % sizeof(int32_t) != 0 ||
      !element_aligned(d->log_decay, d->beta) ||
      !aligned16(d->queries, d->keys, d->values, d->offsets, d->slot_ids, accepted, pool,
                 outputs)) {
    return kStatusInvalidArgument;
  }
  const uint64_t blocks = static_cast<uint64_t>(d->requests) * d->value_heads;
  if (blocks > kMaxGrid) return kStatusInvalidArgument;
  if (d->tokens == 0) return kStatusOk;  // every tree is empty
  const DraftArgs args{d->queries, d->keys, d->values, d->log_decay, d->beta, d->query_stride,
                       d->key_stride, d->value_stride, d->parents, d->offsets, d->slot_ids,
                       accepted, pool, outputs, d->tokens, slots, d->value_heads,
                       d->value_heads / d->key_heads, d->max_nodes, d->scale, d->normalize};
  const auto kernel = pool_dtype == kDtypeF32 ? draft_kernel<float, kCommit>
                                              : draft_kernel<bf16_bits, kCommit>;
  return launch(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kDim), stream, args);
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
