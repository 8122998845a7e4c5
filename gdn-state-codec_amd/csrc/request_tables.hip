// Tables of a ragged batch, from its request lengths, in one launch.
//
// With t_r the tokens of request r (its length, at least 0, cut off where the
// running sum reaches max_tokens) and c_r = ceil(t_r / 64):
//   offsets[r] = t_0 + .. + t_(r-1),  chunk_offsets[r] = c_0 + .. + c_(r-1),
//   chunk row i belongs to the last r with chunk_offsets[r] <= i,
//   order's place of r = #{s : c_s > c_r, or c_s = c_r and s < r}.
//
// What bounds it is the launch: a batch's lengths are at most 16 KB.  Every
// workgroup therefore forms both prefix sums again in its own LDS (16 values a
// thread, one wave scan and one join each) instead of waiting for another
// workgroup, and then writes its 256 chunk rows and places its 16 requests: a
// row finds its request by bisection of the chunk sums, and a request's place is
// counted by 16 lanes over the chunk counts.  24 requests take 4 us, 4096 16 us (of
// which the count of 4096 x 4096 pairs is most; read one at a time it took 28).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gdn_state_codec_layer.h"
#include "lane_exchange.h"
#include "launch.h"

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = GDN_STATE_CODEC_MAX_REQUESTS;
constexpr int kChunk = GDN_STATE_CODEC_CHUNK;
constexpr int kOrderPerBlock = 16;  // requests placed by a workgroup, 16 lanes each

// Sum of the threads before this one; `total` is the workgroup's.
__device__ __forceinline__ int64_t prefix(int64_t x, int64_t (&waves)[4], int64_t& total) {
  const int lane = threadIdx.x & 63;
  int64_t sum = x;
#pragma unroll
  for (int step = 1; step < 64; step <<= 1) {
    const int64_t other = __shfl_up(sum, step);
    if (lane >= step) sum += other;
  }
  __syncthreads();  // the last call's values are read
  if (lane == 63) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 6)) before += waves[w];
    total += waves[w];
  }
  return before + sum - x;
}

__global__ __launch_bounds__(kThreads) void request_tables_kernel(
    const int32_t* __restrict__ lengths, const int32_t* __restrict__ slot_ids, uint32_t requests,
    uint32_t max_tokens, uint32_t rows, int32_t* __restrict__ offsets,
    int32_t* __restrict__ chunk_offsets, int4* __restrict__ chunks, int32_t* __restrict__ order) {
  __shared__ int32_t token_sum[kMaxRequests + 1];
  __shared__ int32_t chunk_sum[kMaxRequests + 1];
  __shared__ int64_t waves[4];
  const int t = threadIdx.x;
  const uint32_t each = (requests + kThreads - 1) / kThreads;  // consecutive requests a thread
  const uint32_t first = min(t * each, requests);
  const uint32_t last = min(first + each, requests);

  // Token sums, cut off at max_tokens (64-bit: 4096 lengths of up to 2^31 - 1).  The
  // lengths are all asked for before the first is used.
  int32_t own[kMaxRequests / kThreads];
#pragma unroll
  for (int i = 0; i < kMaxRequests / kThreads; ++i) {
    own[i] = lengths[min(first + i, requests - 1)];
  }
  int64_t sum = 0;
#pragma unroll
  for (int i = 0; i < kMaxRequests / kThreads; ++i) {
    own[i] = first + i < last ? max(own[i], 0) : 0;
    sum += own[i];
  }
  int64_t total;
  int64_t at = prefix(sum, waves, total);
  const int64_t most = max_tokens;
  int64_t count = 0;
#pragma unroll
  for (int i = 0; i < kMaxRequests / kThreads; ++i) {
    const int64_t begin = min(at, most);
    at += own[i];
    own[i] = static_cast<int32_t>((min(at, most) - begin + kChunk - 1) / kChunk);
    count += own[i];
    if (first + i < last) token_sum[first + i] = static_cast<int32_t>(begin);
  }
  if (t == 0) token_sum[requests] = static_cast<int32_t>(min(total, most));
  int64_t chunk = prefix(count, waves, total);  // its barriers publish token_sum
#pragma unroll
  for (int i = 0; i < kMaxRequests / kThreads; ++i) {
    if (first + i < last) chunk_sum[first + i] = static_cast<int32_t>(chunk);
    chunk += own[i];
  }
  if (t == 0) chunk_sum[requests] = static_cast<int32_t>(total);
  __syncthreads();

  if (blockIdx.x == 0) {
    for (uint32_t r = t; r <= requests; r += kThreads) {
      offsets[r] = token_sum[r];
      chunk_offsets[r] = chunk_sum[r];
    }
  }

  const uint32_t row = blockIdx.x * kThreads + t;
  if (row < rows) {
    int4 entry = make_int4(-1, 0, 0, -1);
    if (row < static_cast<uint32_t>(chunk_sum[requests])) {
      // The last request that starts at or before the row: empty requests
      // before it share its chunk sum and come earlier.
      uint32_t low = 0, high = requests;
      while (high - low > 1) {
        const uint32_t middle = (low + high) / 2;
        if (static_cast<uint32_t>(chunk_sum[middle]) <= row) low = middle;
        else high = middle;
      }
      const int begin = token_sum[low] + (static_cast<int>(row) - chunk_sum[low]) * kChunk;
      entry = make_int4(static_cast<int>(low), begin, min(kChunk, token_sum[low + 1] - begin),
                        slot_ids[low]);
    }
    chunks[row] = entry;
  }

  const uint32_t r = blockIdx.x * kOrderPerBlock + (t >> 4);
  if (r < requests) {  // the same for the 16 lanes of a request
    const int mine = chunk_sum[r + 1] - chunk_sum[r];
    int before = 0;
#pragma unroll 8
    for (uint32_t s = t & 15; s < requests; s += 16) {
      const int other = chunk_sum[s + 1] - chunk_sum[s];
      before += other > mine || (other == mine && s < r) ? 1 : 0;
    }
    before += dpp_xor<1>(before);
    before += dpp_xor<2>(before);
    before += dpp_xor<4>(before);
    before += dpp_xor<8>(before);
    if ((t & 15) == 0) order[before] = static_cast<int32_t>(r);
  }
}

}  // namespace
}  // namespace gdn

extern "C" int32_t statecentric_gdn_state_codec_request_tables_launch_v1(
    void* stream, const int32_t* lengths, const int32_t* slot_ids, uint32_t requests,
    uint32_t max_tokens, uint32_t rows, int32_t* offsets, int32_t* chunk_offsets,
    int32_t* chunks, int32_t* order) {
  if (!lengths || !slot_ids || !offsets || !chunk_offsets || !chunks || !order ||
      requests == 0 || requests > GDN_STATE_CODEC_MAX_REQUESTS || max_tokens > 0x7FFFFFFFu ||
      rows != max_tokens / GDN_STATE_CODEC_CHUNK + requests ||
      !gdn::aligned16(lengths, slot_ids, offsets, chunk_offsets, chunks, order)) {
    return gdn::kStatusInvalidArgument;
  }
  const uint32_t for_rows = (rows + gdn::kThreads - 1) / gdn::kThreads;
  const uint32_t for_order = (requests + gdn::kOrderPerBlock - 1) / gdn::kOrderPerBlock;
  return gdn::launch(gdn::request_tables_kernel, dim3(for_rows > for_order ? for_rows : for_order),
                     dim3(gdn::kThreads), stream, lengths, slot_ids, requests, max_tokens, rows,
                     offsets, chunk_offsets, reinterpret_cast<int4*>(chunks), order);
}
