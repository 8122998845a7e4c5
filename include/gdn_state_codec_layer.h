/*
 * C-ABI of the dense operators around the encoded state on MI355X (gfx950):
 * what a gated-delta-net layer runs before a state is encoded and where a
 * request is not served from an encoded one.
 *
 *   request_tables          tables of a ragged batch from its request lengths
 *   gated_delta_step        one token of the gated delta rule per request, on a
 *                           slot-indexed dense state pool
 *   gated_delta_prefill     the rule over whole ragged sequences, on the pool
 *   gated_delta_forward,
 *   gated_delta_backward    the rule over packed sequences with every gradient
 *   gated_norm, residual_norm (and _backward)
 *                           the norms after and before the block
 *
 * The rule, for one value head with state S [value][key] and a token's
 * q, k (128 keys), v (128 values), log decay g and write strength b:
 *   S <- exp(g) S;   e = v - S k;   S <- S + b e k^T;   o = S q
 * where, with `normalize`, q and k are first divided by
 * sqrt(sum of squares + 1e-6), and q is multiplied by `scale`.  Value head h
 * reads key head h / (value_heads / key_heads).
 *
 * States and their gradients are formed in fp32 throughout.  In the whole-sequence
 * calls an output is a sum over its chunk's start state and the writes since, whose
 * terms are good to 2^-15 each before the sum is rounded to bf16: an output far below
 * its terms (under 2^-6 of them) has fewer bits than bf16 holds.  A NaN or an infinity
 * in a token may reach its request's outputs from its 64-token chunk's start on; other
 * requests never see it.
 *
 * Same conventions as gdn_state_codec_kernel.h: asynchronous on `stream` (NULL
 * = HIP's null stream), no allocation, status 0 / 1 (bad argument) / 5 (launch
 * failed), and every device pointer 16-byte aligned but log_decay and beta, which
 * need their element's alignment only (a slice of a batch may start anywhere).
 */
#ifndef GDN_STATE_CODEC_LAYER_H
#define GDN_STATE_CODEC_LAYER_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations, residual streams and state pools. */
#define GDN_STATE_CODEC_LAYER_F32 0u
#define GDN_STATE_CODEC_LAYER_BF16 1u

/* Tokens of a chunk of the rule's long form, and of a row of `chunks`. */
#define GDN_STATE_CODEC_CHUNK 64u
#define GDN_STATE_CODEC_MAX_REQUESTS 4096u

/* Tables of a ragged batch whose requests' tokens are packed one after another.
 * lengths, slot_ids int32 [requests] (1..4096); a negative length counts as 0,
 * and tokens past max_tokens (<= 2^31 - 1) are cut off.  Writes, all int32:
 *   offsets [requests + 1]        first token of each request, then their total
 *   chunk_offsets [requests + 1]  first row of each request in `chunks`
 *   chunks [rows][4]              {request, first token, tokens 1..64, slot} of
 *                                 each 64-token chunk; past the last chunk
 *                                 {-1, 0, 0, -1}
 *   order [requests]              requests by falling chunk count, equal ones in
 *                                 their own order
 * rows must be max_tokens / 64 + requests: what any lengths need at most. */
int32_t statecentric_gdn_state_codec_request_tables_launch_v1(
    void* stream, const int32_t* lengths, const int32_t* slot_ids,
    uint32_t requests, uint32_t max_tokens, uint32_t rows, int32_t* offsets,
    int32_t* chunk_offsets, int32_t* chunks, int32_t* order);

/* One token per request.  queries, keys bf16 [batch][key_heads][128] and values
 * bf16 [batch][value_heads][128], each with its own distance between tokens
 * (elements, a multiple of 8); log_decay fp32 and beta bf16
 * [batch][value_heads]; pool [slots][value_heads][128 value][128 key] of
 * pool_dtype, updated in place at slot_ids int32 [batch] (distinct); outputs
 * bf16 [batch][value_heads][128].  An entry whose slot id is outside
 * 0..slots-1 (padding, -1) is skipped and its output left as it was. */
int32_t statecentric_gdn_state_codec_gated_delta_step_launch_v1(
    void* stream, const uint16_t* queries, const uint16_t* keys,
    const uint16_t* values, const float* log_decay, const uint16_t* beta,
    void* pool, const int32_t* slot_ids, uint16_t* outputs, uint32_t batch,
    uint32_t slots, uint32_t value_heads, uint32_t key_heads,
    uint64_t query_stride, uint64_t key_stride, uint64_t value_stride,
    uint32_t pool_dtype, float scale, uint32_t normalize);

/* A packed ragged batch and the scratch its whole-sequence form works in.  Where
 * tokens is 0, every pointer to rows of tokens, here and in the calls, may be NULL:
 * each request is then empty. */
typedef struct gdn_state_codec_rule {
  const uint16_t* queries;      /* bf16 [tokens][key_heads][128] */
  const uint16_t* keys;         /* bf16 [tokens][key_heads][128] */
  const uint16_t* values;       /* bf16 [tokens][value_heads][128] */
  const float* log_decay;       /* [tokens][value_heads] */
  const uint16_t* beta;         /* bf16 [tokens][value_heads] */
  uint64_t query_stride;        /* elements between tokens, multiples of 8 */
  uint64_t key_stride;
  uint64_t value_stride;
  const int32_t* offsets;       /* request_tables' outputs for max_tokens = tokens */
  const int32_t* chunk_offsets;
  const int32_t* chunks;
  const int32_t* order;
  void* workspace;              /* gated_delta_workspace(...) bytes at least */
  uint64_t workspace_bytes;
  uint32_t requests;            /* 1..4096 */
  uint32_t rows;                /* tokens / 64 + requests */
  uint32_t tokens;
  uint32_t value_heads;
  uint32_t key_heads;
  float scale;
  uint32_t normalize;
} gdn_state_codec_rule;

/* Bytes of the workspace: for prefill (train 0), or for a forward and backward
 * pass (train 1; the backward pass reads what the forward pass left there). */
uint64_t statecentric_gdn_state_codec_gated_delta_workspace_v1(
    uint32_t rows, uint32_t value_heads, uint32_t key_heads, uint32_t train);

/* Whole sequences on a slot-indexed pool [slots][value_heads][128 value]
 * [128 key] of pool_dtype (the tables made with the same slot ids): request r starts from its slot's state (resume NULL or
 * resume[r] != 0) or from zeros, and leaves its final state there.  slot_ids int32
 * [requests] (distinct); a request whose slot is outside 0..slots-1 (padding, -1)
 * is skipped, its outputs left as they were.  An empty request leaves its state, or
 * zeros where it does not resume.  outputs bf16 [tokens][value_heads][128]. */
int32_t statecentric_gdn_state_codec_gated_delta_prefill_launch_v1(
    void* stream, const gdn_state_codec_rule* rule, const int32_t* slot_ids,
    const int32_t* resume, void* pool, uint32_t slots, uint32_t pool_dtype,
    uint16_t* outputs);

/* Whole packed sequences for training: initial (or NULL: zeros) and final_states
 * fp32 [requests][value_heads][128 value][128 key]; the tables' slots are not
 * read.  Outputs of tokens of no request are zeros.  Leaves in the workspace what
 * the backward pass reads. */
int32_t statecentric_gdn_state_codec_gated_delta_forward_launch_v1(
    void* stream, const gdn_state_codec_rule* rule, const float* initial,
    float* final_states, uint16_t* outputs);

/* Gradients of gated_delta_forward, from d_outputs (bf16, contiguous) and d_final
 * (or NULL: zeros), with the same `rule` and its workspace as that call left it:
 * d_queries, d_keys bf16 [tokens][key_heads][128], d_values bf16
 * [tokens][value_heads][128], d_log_decay fp32 and d_beta bf16
 * [tokens][value_heads], d_initial (or NULL) like initial.  Gradients of tokens of
 * no request are zeros.  May be called again. */
int32_t statecentric_gdn_state_codec_gated_delta_backward_launch_v1(
    void* stream, const gdn_state_codec_rule* rule, const uint16_t* d_outputs,
    const float* d_final, uint16_t* d_queries, uint16_t* d_keys, uint16_t* d_values,
    float* d_log_decay, uint16_t* d_beta, float* d_initial);

/* out = x / sqrt(mean(x^2) + eps) * weight * gate * sigmoid(gate) over rows of
 * 128.  x, gate, out [rows][128] of `dtype`, weight fp32 [128]. */
int32_t statecentric_gdn_state_codec_gated_norm_launch_v1(
    void* stream, const void* x, const void* gate, const float* weight, void* out,
    uint64_t rows, uint32_t dtype, float eps);

/* Its gradients: d_x, d_gate [rows][128] of `dtype`, d_weight fp32 [128].
 * partials: fp32 [norm_partials(rows, 128)][128] scratch. */
int32_t statecentric_gdn_state_codec_gated_norm_backward_launch_v1(
    void* stream, const void* x, const void* gate, const float* weight,
    const void* d_out, void* d_x, void* d_gate, float* d_weight, float* partials,
    uint64_t rows, uint32_t dtype, float eps);

/* sum = residual + scale * x (rounded to the stream's type), and
 * out = sum / sqrt(mean(sum^2) + eps) * weight over rows of `width` (a multiple
 * of 8, up to 16384).  x, out [rows][width] of `dtype`; residual, sum
 * [rows][width] of `stream_dtype` (sum may be residual itself); weight fp32. */
int32_t statecentric_gdn_state_codec_residual_norm_launch_v1(
    void* stream, const void* x, const void* residual, const float* weight,
    void* out, void* sum, uint64_t rows, uint32_t width, uint32_t dtype,
    uint32_t stream_dtype, float scale, float eps);

/* Its gradients from d_out (`dtype`) and d_sum (`stream_dtype`, or NULL for
 * zeros): d_residual of `stream_dtype`, d_x = scale * d_residual of `dtype`
 * (each rounded once), d_weight fp32 [width].  partials: fp32
 * [norm_partials(rows, width)][width] scratch. */
int32_t statecentric_gdn_state_codec_residual_norm_backward_launch_v1(
    void* stream, const void* sum, const float* weight, const void* d_out,
    const void* d_sum, void* d_x, void* d_residual, float* d_weight,
    float* partials, uint64_t rows, uint32_t width, uint32_t dtype,
    uint32_t stream_dtype, float scale, float eps);

/* Rows of the backward passes' partials scratch. */
uint32_t statecentric_gdn_state_codec_norm_partials_v1(uint64_t rows, uint32_t width);

#ifdef __cplusplus
}
#endif

#endif /* GDN_STATE_CODEC_LAYER_H */
