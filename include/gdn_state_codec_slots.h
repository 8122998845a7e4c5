/*
 * C-ABI of the slots of a state cache on MI355X (gfx950): copying, forking and
 * reordering them, clearing freed ones, and packing the live ones to the front.
 *
 *   slot_moves        the order in which pairs (source, target) can be copied in place
 *   compaction_moves  the pairs that pack live slots to the front
 *   copy_slots        the copies themselves, over any buffers that hold a row a slot:
 *                     dense pools of some layers, the buffers of encoded slots
 *
 * Same conventions as gdn_state_codec_kernel.h: asynchronous on `stream` (NULL
 * = HIP's null stream), no allocation, status 0 / 1 (bad argument) / 5 (launch
 * failed), and every device pointer 16-byte aligned but copy_slots' buffers.
 */
#ifndef GDN_STATE_CODEC_SLOTS_H
#define GDN_STATE_CODEC_SLOTS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GDN_STATE_CODEC_MAX_MOVES 4096u
#define GDN_STATE_CODEC_MAX_COMPACTED 65536u

/* Rows of `steps`, in an order in which they can be carried out one after another:
 *   {source, target, flags, end}   all int32
 * source -1: zeros; target -1: nothing; end: the row behind the last that this one has
 * to be carried out in turn with. */
#define GDN_STATE_CODEC_MOVE_SAVES 1u  /* first keep what the target holds */
#define GDN_STATE_CODEC_MOVE_SAVED 2u  /* the source is what was kept */

/* steps [pairs][4] of the copies targets[i] <- sources[i] (int32 [pairs], 1..4096), all
 * of them at once: a source is what it held before any copy, in chains and in cycles too.
 * A source of -1 clears its target.  A pair whose target, or any other source, is outside
 * 0..slots-1 is left out (padding); of pairs with one target the last counts. */
int32_t statecentric_gdn_state_codec_slot_moves_launch_v1(
    void* stream, const int32_t* sources, const int32_t* targets, uint32_t pairs,
    uint32_t slots, int32_t* steps);

/* The moves that bring the live slots (live[i] != 0, int32 [slots], 1..65536 slots) into
 * the first `count` places: the k-th live slot from place `count` on goes to the k-th
 * free one before it.  steps [(slots + 1) / 2][4]; placed int32 [slots]: each live slot's
 * new place, -1 for others; count int32 [1]: live slots. */
int32_t statecentric_gdn_state_codec_compaction_moves_launch_v1(
    void* stream, const int32_t* live, uint32_t slots, int32_t* steps, int32_t* placed,
    int32_t* count);

/* One tensor of a cache: `bytes` a slot, slots side by side.  `to` is `from` itself, or
 * other memory; what one buffer writes overlaps nothing that another reads or writes. */
typedef struct gdn_state_codec_slot_buffer {
  const void* from;
  void* to;
  uint64_t bytes;
} gdn_state_codec_slot_buffer;

/* to[target] <- from[source] for every row of `steps` (of slot_moves or compaction_moves
 * for the same number of slots) and every one of `count` buffers (host memory, read before
 * the call returns). */
int32_t statecentric_gdn_state_codec_copy_slots_launch_v1(
    void* stream, const gdn_state_codec_slot_buffer* buffers, uint32_t count,
    const int32_t* steps, uint32_t rows, uint32_t slots);

#ifdef __cplusplus
}
#endif

#endif /* GDN_STATE_CODEC_SLOTS_H */
