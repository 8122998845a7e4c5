"""MI355X (gfx950) GDN state codec: int8 codec of Qwen3.5 gated-delta-net
recurrent-state head tiles, the encoded projection, the windowed decode step,
its window-boundary refit and the LQCAPS01 capsule wire format, behind the
reference's ``statecentric_gdn_state_codec_*`` C-ABI; and the dense operators of a
gated-delta-net layer around that state (``layer``) and moves between its slots
(``slots``)."""

from ._native import NativeLibrary, library_dir, library_path, native
from .codec import (
    LAYOUT_KEY_VALUE,
    LAYOUT_VALUE_KEY,
    decode,
    encode,
    pool_decode,
    pool_encode,
    project_chunked,
    project_decode,
)
from .capsule import CapsuleIdentity
from .layer import (
    RequestTables,
    gated_delta_commit,
    gated_delta_prefill,
    gated_delta_rule,
    gated_delta_step,
    gated_delta_tree,
    gated_norm,
    request_tables,
    residual_norm,
)
from .runtime import GdnStateCodecExperiment, GdnStateCodecRuntime
from .slots import Compaction, SlotMoves, compaction_moves, copy_slots, slot_moves
from .window import DecodeRuntime, WindowSlot

__all__ = [
    "CapsuleIdentity",
    "Compaction",
    "LAYOUT_KEY_VALUE",
    "LAYOUT_VALUE_KEY",
    "DecodeRuntime",
    "RequestTables",
    "GdnStateCodecExperiment",
    "GdnStateCodecRuntime",
    "SlotMoves",
    "WindowSlot",
    "NativeLibrary",
    "compaction_moves",
    "copy_slots",
    "decode",
    "encode",
    "gated_delta_commit",
    "gated_delta_prefill",
    "gated_delta_rule",
    "gated_delta_step",
    "gated_delta_tree",
    "gated_norm",
    "library_dir",
    "library_path",
    "native",
    "pool_decode",
    "pool_encode",
    "project_chunked",
    "project_decode",
    "request_tables",
    "residual_norm",
    "slot_moves",
]
