// The sequential half of the gated delta rule's chunked form, forward
// (formulas, layouts and precision in delta_chunk.h).
//
// Column v of a state [key][value] meets only column v of V, E and O, so one
// wavefront takes 16 kColumns columns of one request's value head through all its
// chunks, with the state in its accumulators: no LDS, no barrier, no exchange
// between lanes.  Per chunk and 16 columns it issues
//   K S0: 48, N (b R): 36, P (b E): 18, Q S0: 32, K^T U: 48   matrix instructions
// (K S0's results are the operand of N, N's of both updates, so S0 to S1 is one
// chain).  The operands come from the workspace in the order the lanes hold them,
// 16 bytes a lane and load.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "delta_chunk.h"

namespace gdn {

int32_t launch_delta_prepare(void* stream, const RuleArgs& args, bf16_bits* outputs);

struct ScanArgs {
  RuleArgs rule;
  const void* initial;       // states [..][value head][value][key], or null: zeros
  void* final_states;        // may be `initial`
  const int32_t* slot_ids;   // of each request, or null: the request's own place
  const int32_t* resume;     // 0: start from zeros, or null: all resume
  uint32_t slots;
  bf16_bits* outputs;        // [tokens][value head][128]
};

namespace {

// A chunk's operands in LDS: K, Q and K^T of the key head, then the first 32 KiB
// of the value head's block (factors, N, P b; 512 bytes of it are not used).
constexpr int kKeyStage = 3 * kKeyTiles * kTileBytes;
constexpr int kValueStage = 32 * kTileBytes;
constexpr int kStage = kKeyStage + kValueStage;
static_assert(value_block_bytes(false) <= kValueStage, "the stage holds a value block");
static_assert(2 * kStage <= static_cast<int>(kLdsPerCu), "two stages fill the LDS");

template <int kWaves>
__device__ __forceinline__ void stage_chunk(const char* keys, const char* block, int wave,
                                            int lane, uint32_t to) {
#pragma unroll
  for (int i = 0; i < 80 / kWaves; ++i) {
    const int tile = i * kWaves + wave;
    const char* from = tile < 48 ? keys + tile * kTileBytes : block + (tile - 48) * kTileBytes;
    stage_tile(from, lane, to + tile * kTileBytes);
  }
}

template <typename Pool, int kWaves, bool kTrain>
__global__ __launch_bounds__(64 * kWaves, 1) void delta_scan_kernel(ScanArgs args) {
  constexpr int kSlices = kDim / (16 * kWaves);
  __shared__ __align__(16) char stages[2][kStage];
  const RuleArgs& a = args.rule;
  const ChunkSpace& space = a.space;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  // A head's slices share their operands: they get consecutive places of one XCD
  // (the dispatcher deals workgroups out to the 8 XCDs in turn).
  const uint32_t turn = blockIdx.x >> 3;
  const uint64_t item = static_cast<uint64_t>(turn / kSlices) * 8 + (blockIdx.x & 7);
  if (item >= static_cast<uint64_t>(a.requests) * space.value_heads) return;
  const uint32_t head = static_cast<uint32_t>(item % space.value_heads);
  const int32_t request = a.order[item / space.value_heads];
  if (request < 0 || static_cast<uint32_t>(request) >= a.requests) return;
  const int value = (turn % kSlices) * 16 * kWaves + 16 * wave + r;  // this lane's column
  const int32_t slot = args.slot_ids ? args.slot_ids[request] : request;
  if (slot < 0 || static_cast<uint32_t>(slot) >= args.slots) return;  // padding
  const uint64_t tile = (static_cast<uint64_t>(slot) * space.value_heads + head) * kTile +
                        value * kDim + 4 * g;

  f32x4 state[8];  // keys 16 t + 4 g + i
  const bool resumed = args.initial && (!args.resume || args.resume[request] != 0);
#pragma unroll
  for (int t = 0; t < 8; ++t) state[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (resumed) {
    const Pool* p = static_cast<const Pool*>(args.initial) + tile;
#pragma unroll
    for (int t = 0; t < 8; ++t) state[t] = load_cells(p + 16 * t);
  }

  // The request's tokens and chunk rows, as far as the tables stay inside the batch.
  const uint32_t first_row = min(static_cast<uint32_t>(a.chunk_offsets[request]), space.rows);
  const uint32_t rows = min(static_cast<uint32_t>(a.chunk_offsets[request + 1]), space.rows) -
                        first_row;
  const uint32_t begin = min(static_cast<uint32_t>(a.offsets[request]), a.tokens);
  const uint32_t length = min(static_cast<uint32_t>(a.offsets[request + 1]), a.tokens) - begin;
  const uint32_t chunks = min(rows, (length + kChunk - 1) / kChunk);
  const uint32_t stage_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) char*)&stages[0][0]));
  const uint64_t token_step = static_cast<uint64_t>(space.value_heads) * kDim;

  bf16_bits values[4][4];  // of the tokens 16 t + 4 g + i
  const auto fetch = [&](uint32_t c) {
    const int last = min(static_cast<int>(length - c * kChunk), kChunk) - 1;
    stage_chunk<kWaves>(space.key_block(first_row + c, head / a.group),
                        space.value_block(first_row + c, head), wave, lane,
                        stage_at + (c & 1) * kStage);
    const bf16_bits* v = a.values + static_cast<uint64_t>(begin + c * kChunk) * a.value_stride +
                         head * kDim + value;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        values[t][i] = v[min(16 * t + 4 * g + i, last) * a.value_stride];
      }
    }
  };
  if (chunks != 0) fetch(0);

  f32x4 error[4], out[4];
  const auto store_outputs = [&](uint32_t c, int tokens) {
    if constexpr (kTrain) {
      float* e = space.errors(first_row + c, head) + value;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[(16 * t + 4 * g + i) * kDim] = error[t][i];
      }
    }
    bf16_bits* o = args.outputs + (begin + c * kChunk) * token_step + head * kDim + value;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int token = 16 * t + 4 * g + i;
        if (token < tokens) {
          o[token * token_step] = static_cast<bf16_bits>(bf16_pair(out[t][i], 0.0f));
        }
      }
    }
  };

  for (uint32_t c = 0; c < chunks; ++c) {
    stage_ready();
    const uint32_t row = first_row + c;
    const char* const keys = stages[c & 1];
    const char* const block = keys + kKeyStage;
    const uint4* const k_rows = reinterpret_cast<const uint4*>(keys + kKeyRows) + lane;
    const uint4* const q_rows = reinterpret_cast<const uint4*>(keys + kQueryRows) + lane;
    const uint4* const k_columns = reinterpret_cast<const uint4*>(keys + kKeyColumns) + lane;
    const uint4* const solve = reinterpret_cast<const uint4*>(block + kSolve) + lane;
    const uint4* const read_out = reinterpret_cast<const uint4*>(block + kReadOut) + lane;
    const float* const factors = reinterpret_cast<const float*>(block) + 4 * g;
    const int tokens = min(static_cast<int>(length - c * kChunk), kChunk);
    f32x4 value_rows[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        value_rows[t][i] = 16 * t + 4 * g + i < tokens ? widen(values[t][i]) : 0.0f;
        // Used before the next loads are issued, so that no wait for it covers them.
        asm volatile("" : "+v"(value_rows[t][i]));
      }
    }
    // The next chunk's loads and the last one's stores have this chunk's products
    // to finish in.
    if (c + 1 < chunks) fetch(c + 1);
    if (c != 0) store_outputs(c - 1, kChunk);  // only the last chunk can be short
    if constexpr (kTrain) {
      float* p = space.state(row, head) + value;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[(16 * t + 4 * g + i) * kDim] = state[t][i];
      }
    }

    {
      uint4 part[4][3];  // of the state, over the keys
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        split3(state[2 * step], state[2 * step + 1], part[step]);
      }
      // R = V - exp(G) K S0
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 seen = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          seen = mfma3(k_rows[(4 * t + step) * 64], part[step], seen);
        }
        const f32x4 factor = load4(factors + kReadKey * kChunk + 16 * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) error[t][i] = fmaf(-factor[i], seen[i], value_rows[t][i]);
      }
      // exp(G) Q S0, from two of the state's parts: 2^-15 of terms whose sums
      // become bf16 outputs.
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 read = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          const uint4 q = q_rows[(4 * t + step) * 64];
          read = mfma(q, part[step][1], read);
          read = mfma(q, part[step][0], read);
        }
        const f32x4 factor = load4(factors + kReadQuery * kChunk + 16 * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) out[t][i] = factor[i] * read[i];
      }
    }
    // E = R + N (b R)
    {
      uint4 part[2][3];
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        f32x4 x[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x4 b = load4(factors + kStrength * kChunk + 32 * step + 16 * u);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[u][i] = b[i] * error[2 * step + u][i];
        }
        split3(x[0], x[1], part[step]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int step = 0; step < lower_steps(t); ++step) {
          uint4 n[3];
#pragma unroll
          for (int p = 0; p < 3; ++p) n[p] = solve[(p * kTriangle + lower_tile(t, step)) * 64];
          error[t] = mfma6(n, part[step], error[t]);
        }
      }
    }
    // S1 = exp(G_63) S0 + K^T (write b E), and O += (P b) E
    const float whole = factors[kWhole * kChunk];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) state[t][i] *= whole;
    }
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      uint4 written[3], plain[3];
      f32x4 x[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f32x4 b = load4(factors + kStrength * kChunk + 32 * step + 16 * u);
        const f32x4 w = load4(factors + kWrite * kChunk + 32 * step + 16 * u);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[u][i] = w[i] * (b[i] * error[2 * step + u][i]);
      }
      split3(x[0], x[1], written);
      split3(error[2 * step], error[2 * step + 1], plain);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        state[t] = mfma3(k_columns[(2 * t + step) * 64], written, state[t]);
      }
#pragma unroll
      for (int t = 2 * step; t < 4; ++t) {  // rows 0..31 end in step 0
        const int place = lower_tile(t, step);
        const uint4 high = read_out[place * 64], low = read_out[(kTriangle + place) * 64];
        out[t] = mfma(low, plain[0], out[t]);
        out[t] = mfma(high, plain[1], out[t]);
        out[t] = mfma(high, plain[0], out[t]);
      }
    }
  }
  if (chunks != 0) store_outputs(chunks - 1, length - (chunks - 1) * kChunk);

  Pool* p = static_cast<Pool*>(args.final_states) + tile;
#pragma unroll
  for (int t = 0; t < 8; ++t) store_cells(p + 16 * t, state[t]);
}

template <typename Pool, int kWaves, bool kTrain>
int32_t launch_scan(void* stream, const ScanArgs& args) {
  constexpr uint64_t kSlices = kDim / (16 * kWaves);
  const uint64_t items = static_cast<uint64_t>(args.rule.requests) * args.rule.space.value_heads;
  const uint64_t blocks = (items + 7) / 8 * 8 * kSlices;
  if (blocks > kMaxGrid) return kStatusInvalidArgument;
  return launch(delta_scan_kernel<Pool, kWaves, kTrain>, dim3(static_cast<uint32_t>(blocks)),
                dim3(64 * kWaves), stream, args);
}

}  // namespace

int32_t launch_delta_scan(void* stream, const ScanArgs& args, uint32_t dtype) {
  if (args.rule.space.train) return launch_scan<float, 4, true>(stream, args);
  return dtype == kDtypeF32 ? launch_scan<float, 4, false>(stream, args)
                            : launch_scan<bf16_bits, 4, false>(stream, args);
}

// Checks the caller's arguments and fills the kernels'; false: a bad argument.
bool rule_args(const gdn_state_codec_rule* rule, bool train, RuleArgs& a) {
  if (!rule || !rule->queries || !rule->keys || !rule->values || !rule->log_decay ||
      !rule->beta || !rule->offsets || !rule->chunk_offsets || !rule->chunks || !rule->order ||
      !rule->workspace || rule->requests == 0 || rule->requests > GDN_STATE_CODEC_MAX_REQUESTS ||
      rule->tokens > 0x7FFFFFFFu || rule->rows != rule->tokens / kChunk + rule->requests ||
      rule->key_heads == 0 || rule->value_heads == 0 ||
      rule->value_heads % rule->key_heads != 0 || rule->normalize > 1 ||
      rule->query_stride % 8 != 0 || rule->key_stride % 8 != 0 || rule->value_stride % 8 != 0 ||
      static_cast<uint64_t>(rule->rows) * rule->value_heads > kMaxGrid ||
      !aligned16(rule->queries, rule->keys, rule->values, rule->log_decay, rule->beta,
                 rule->offsets, rule->chunk_offsets, rule->chunks, rule->order,
                 rule->workspace)) {
    return false;
  }
  a = RuleArgs{rule->queries, rule->keys, rule->values, rule->log_decay, rule->beta,
               rule->query_stride, rule->key_stride, rule->value_stride, rule->offsets,
               rule->chunk_offsets, reinterpret_cast<const int4*>(rule->chunks), rule->order,
               rule->requests, rule->tokens, rule->value_heads / rule->key_heads, rule->scale,
               rule->normalize,
               ChunkSpace{static_cast<char*>(rule->workspace), rule->rows, rule->key_heads,
                          rule->value_heads, train}};
  return rule->workspace_bytes >= a.space.total();
}

}  // namespace gdn

extern "C" uint64_t statecentric_gdn_state_codec_gated_delta_workspace_v1(
    uint32_t rows, uint32_t value_heads, uint32_t key_heads, uint32_t train) {
  return gdn::ChunkSpace{nullptr, rows, key_heads, value_heads, train != 0}.total();
}

extern "C" int32_t statecentric_gdn_state_codec_gated_delta_prefill_launch_v1(
    void* stream, const gdn_state_codec_rule* rule, const int32_t* slot_ids,
    const int32_t* resume, void* pool, uint32_t slots, uint32_t pool_dtype, uint16_t* outputs) {
  gdn::ScanArgs args{};
  if (!gdn::rule_args(rule, false, args.rule) || !slot_ids || !pool || !outputs || slots == 0 ||
      slots > 0x7FFFFFFFu || pool_dtype > gdn::kDtypeBF16 ||
      !gdn::aligned16(slot_ids, resume, pool, outputs)) {
    return gdn::kStatusInvalidArgument;
  }
  args.initial = pool, args.final_states = pool, args.slot_ids = slot_ids, args.resume = resume;
  args.slots = slots, args.outputs = outputs;
  const int32_t status = gdn::launch_delta_prepare(stream, args.rule, outputs);
  return status != gdn::kStatusOk ? status : gdn::launch_delta_scan(stream, args, pool_dtype);
}

extern "C" int32_t statecentric_gdn_state_codec_gated_delta_forward_launch_v1(
    void* stream, const gdn_state_codec_rule* rule, const float* initial, float* final_states,
    uint16_t* outputs) {
  gdn::ScanArgs args{};
  if (!gdn::rule_args(rule, true, args.rule) || !final_states || !outputs ||
      !gdn::aligned16(initial, final_states, outputs)) {
    return gdn::kStatusInvalidArgument;
  }
  args.initial = initial, args.final_states = final_states, args.slots = rule->requests;
  args.outputs = outputs;
  const int32_t status = gdn::launch_delta_prepare(stream, args.rule, outputs);
  return status != gdn::kStatusOk ? status
                                  : gdn::launch_delta_scan(stream, args, gdn::kDtypeF32);
}
