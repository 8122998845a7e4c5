"""torch-facing moves between the slots of a state cache
(include/gdn_state_codec_slots.h): copying, forking and reordering slots, clearing
freed ones, and packing the live ones to the front.

A cache is any set of contiguous tensors whose first dimension is the slot: the dense
pools of some layers, the buffers of encoded slots (:meth:`WindowSlot.slot_rows`).  Which
slots go where stays on the device, and nothing here waits for the GPU.  Checks raise
``RuntimeError``, as the layer operators' do.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Sequence

import torch

from ._native import native
from .layer import _dense, _fail, _launched, _not_differentiated, _on_device, _stream

MAX_MOVES = 4096
MAX_COMPACTED = 65536


class SlotMoves(NamedTuple):
    """Copies between the slots of a cache, in an order in which they can be done."""

    steps: torch.Tensor  # int32 [rows,4]: source, target, flags, end (the C header's)
    slots: int           # of the cache that they are for


class Compaction(NamedTuple):
    """The moves that pack a cache's live slots to the front, and where they go."""

    moves: SlotMoves
    placed: torch.Tensor  # int32 [slots]: each live slot's new place, -1 for others
    count: torch.Tensor   # int32 [1]: live slots, the first places after the moves


def slot_moves(sources: torch.Tensor, targets: torch.Tensor, slots: int) -> SlotMoves:
    """The copies ``targets[i] <- sources[i]`` (device int32 [N], N in 1..4096) between
    the slots 0..``slots``-1 of a cache, all of them at once: a source is what it held
    before, also where another pair overwrites it (a beam search's reordering, swaps).
    A source may go to many targets (a fork), and a source of -1 clears its target (a freed
    slot).  A pair whose target, or any other source, is no slot is left out (padding); of
    pairs with one target the last counts.  Serves any number of :func:`copy_slots` calls."""
    pairs = sources.numel()
    if not 1 <= pairs <= MAX_MOVES:
        _fail(f"slot moves must be 1..{MAX_MOVES} pairs")
    _dense(sources, "source slots", (pairs,), torch.int32)
    _dense(targets, "target slots", (pairs,), torch.int32)
    if not 1 <= slots < 2 ** 31:
        _fail("slot moves need a cache of 1..2^31-1 slots")
    steps = torch.empty((pairs, 4), dtype=torch.int32, device=sources.device)
    _launched(native().slot_moves_launch_v1(
        _stream(), sources.data_ptr(), targets.data_ptr(), pairs, slots, steps.data_ptr()),
        "slot moves")
    return SlotMoves(steps, slots)


def compaction_moves(live: torch.Tensor) -> Compaction:
    """The moves that bring the slots with a nonzero in ``live`` (device int32 [slots],
    1..65536 slots) into the first places: those already there stay, and the k-th live slot
    behind them goes to the k-th free place.  Free slots keep what they hold."""
    slots = live.numel()
    if not 1 <= slots <= MAX_COMPACTED:
        _fail(f"compaction takes 1..{MAX_COMPACTED} slots")
    _dense(live, "live slots", (slots,), torch.int32)
    rows = (slots + 1) // 2
    # One allocation; each table starts on a 16-byte boundary.
    buffer = torch.empty(4 * rows + 4 + slots, dtype=torch.int32, device=live.device)
    steps, count, _, placed = buffer.split_with_sizes((4 * rows, 1, 3, slots))
    _launched(native().compaction_moves_launch_v1(
        _stream(), live.data_ptr(), slots, steps.data_ptr(), placed.data_ptr(),
        count.data_ptr()), "compaction moves")
    return Compaction(SlotMoves(steps.view(rows, 4), slots), placed, count)


def _apart(written, read=()) -> None:
    """Refuses tensors that are written and share memory with another, which the copies
    would race on."""
    ranges = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), writes)
                    for tensors, writes in ((written, True), (read, False)) for t in tensors)
    written_to = read_to = 0
    for begin, end, writes in ranges:
        if begin < written_to or (writes and begin < read_to):
            _fail("slot buffers must not share memory")
        if writes:
            written_to = max(written_to, end)
        else:
            read_to = max(read_to, end)


def copy_slots(buffers: torch.Tensor | Sequence[torch.Tensor], moves: SlotMoves,
               into: torch.Tensor | Sequence[torch.Tensor] | None = None) -> None:
    """Carries ``moves`` out on every tensor of a cache: each contiguous
    [moves.slots, ...], of any types and sizes, sharing no memory.  With ``into``, tensors
    of the same shapes and types, the rows go there from ``buffers``, which stay as they
    are (one may be read into several).  One launch for every 64 tensors."""
    if isinstance(buffers, torch.Tensor):
        buffers = (buffers,)
    if isinstance(into, torch.Tensor):
        into = (into,)
    if not buffers or (into is not None and len(into) != len(buffers)):
        _fail("copying slots takes at least one buffer, and as many to copy into")
    steps, slots = moves
    if steps.dim() != 2 or steps.shape[0] < 1:
        _fail("slot moves must be [rows,4]")
    _dense(steps, "slot moves", (steps.shape[0], 4), torch.int32)
    held = []
    fields = []  # of gdn_state_codec_slot_buffer, one after another
    for i, t in enumerate(buffers):
        if t.dim() < 1 or t.shape[0] != slots or not t.is_contiguous():
            _fail(f"slot buffers must be contiguous [{slots},...], got {tuple(t.shape)} with "
                  f"strides {tuple(t.stride())}")
        _on_device(t, "slot buffer")
        to = t
        if into is not None:
            to = into[i]
            _dense(to, "slot buffer to copy into", t.shape, t.dtype)
        size = t.numel()
        if size:
            held.append((t, to))
            fields += (t.data_ptr(), to.data_ptr(), size // slots * t.element_size())
    _not_differentiated("copying slots", *buffers, *(into or ()))
    if not held:
        return
    if into is not None:
        _apart([to for _, to in held], [t for t, _ in held])
    elif len(held) > 1:
        _apart([t for t, _ in held])
    _launched(native().copy_slots_launch_v1(
        _stream(), (ctypes.c_uint64 * len(fields))(*fields), len(held), steps.data_ptr(),
        steps.shape[0], slots), "copy slots")
