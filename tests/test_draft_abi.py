"""The C-ABI of drafted trees and slot moves, and what their functions refuse, on a machine
without a GPU: bad arguments return 1 before any HIP call."""

from __future__ import annotations

import ctypes
import types

import pytest
import torch

import gdn_state_codec as gdn
from gdn_state_codec import _native, layer, slots
from gdn_state_codec._native import DraftsStruct

P = ctypes.c_void_p(1 << 20)  # 16-byte aligned, never dereferenced
OFF = ctypes.c_void_p((1 << 20) + 4)
TOKEN_POINTERS = ("queries", "keys", "values", "log_decay", "beta", "parents")
TABLES = ("offsets", "slot_ids")


@pytest.fixture(scope="module")
def lib():
    return _native.NativeLibrary()


def drafts(**changes):
    fields = {name: P for name in TOKEN_POINTERS + TABLES}
    fields.update(query_stride=256, key_stride=256, value_stride=512, requests=3, tokens=30,
                  value_heads=4, key_heads=2, max_nodes=64, scale=1.0, normalize=1)
    fields.update(changes)
    return DraftsStruct(**fields)


@pytest.mark.parametrize("entry", ["tree", "commit"])
def test_drafts_admission(lib, entry):
    given = dict(queries=None) if entry == "commit" else {}

    def call(d, pool=P, slots=4, dtype=0, last=P):
        d = None if d is None else ctypes.byref(d)
        if entry == "tree":
            return lib.gated_delta_tree_launch_v1(None, d, pool, slots, dtype, last)
        return lib.gated_delta_commit_launch_v1(None, d, last, pool, slots, dtype)

    assert call(None) == 1
    for name in TOKEN_POINTERS + TABLES:
        if name not in given:
            assert call(drafts(**given, **{name: None})) == 1, name
            off = {"log_decay": 2, "beta": 1, "parents": 2}.get(name, 8)
            moved = ctypes.c_void_p((1 << 20) + off)
            assert call(drafts(**given, **{name: moved})) == 1, name
    for bad in (dict(requests=0), dict(requests=4097), dict(value_heads=3), dict(key_heads=0),
                dict(value_heads=0), dict(normalize=2), dict(max_nodes=0), dict(max_nodes=65),
                dict(query_stride=252), dict(key_stride=4), dict(value_stride=513),
                dict(key_stride=(1 << 24) + 8), dict(value_stride=(1 << 24) + 8),
                dict(query_stride=(1 << 24) + 8), dict(value_heads=(1 << 17) + 1, key_heads=1),
                dict(tokens=1 << 31), dict(value_heads=1 << 17, requests=4096, key_heads=1)):
        assert call(drafts(**{**given, **bad})) == 1, bad
    for bad in (dict(pool=None), dict(pool=OFF), dict(slots=0), dict(slots=1 << 31),
                dict(dtype=2), dict(last=None), dict(last=OFF)):
        assert call(drafts(**given), **bad) == 1, bad
    if entry == "commit":
        assert call(drafts()) == 1  # queries are the tree's


@pytest.mark.parametrize("entry", ["tree", "commit"])
def test_no_tokens_take_no_launch(lib, entry):
    """Every tree is empty, and the token pointers may be null: 0 without a GPU."""
    none = drafts(tokens=0, **{name: None for name in TOKEN_POINTERS})
    if entry == "tree":
        assert lib.gated_delta_tree_launch_v1(None, ctypes.byref(none), P, 4, 0, None) == 0
    else:
        assert lib.gated_delta_commit_launch_v1(None, ctypes.byref(none), P, P, 4, 0) == 0


def test_moves_admission(lib):
    def moves(*p, pairs=4, slots=9):
        return lib.slot_moves_launch_v1(None, p[0], p[1], pairs, slots, p[2])

    def compaction(*p, slots=9):
        return lib.compaction_moves_launch_v1(None, p[0], slots, *p[1:])

    for call, n in ((moves, 3), (compaction, 4)):
        for i in range(n):
            for bad in (None, OFF):
                args = [P] * n
                args[i] = bad
                assert call(*args) == 1, i
    for bad in (dict(pairs=0), dict(pairs=4097), dict(slots=0), dict(slots=1 << 31)):
        assert moves(P, P, P, **bad) == 1, bad
    for bad in (dict(slots=0), dict(slots=65537)):
        assert compaction(P, P, P, P, **bad) == 1, bad


def test_copy_admission(lib):
    def copy(buffers=((1 << 20, 1 << 20, 64),), count=None, steps=P, rows=3, slots=9):
        flat = [x or 0 for buffer in buffers for x in buffer]
        held = (ctypes.c_uint64 * max(3, len(flat)))(*flat)
        count = len(buffers) if count is None else count
        return lib.copy_slots_launch_v1(None, held, count, steps, rows, slots)

    assert lib.copy_slots_launch_v1(None, None, 1, P, 3, 9) == 1
    for bad in (dict(count=0), dict(steps=None), dict(steps=OFF), dict(rows=0),
                dict(rows=1 << 31), dict(slots=0), dict(slots=1 << 31),
                dict(buffers=((None, 1 << 20, 64),)), dict(buffers=((1 << 20, None, 64),)),
                dict(buffers=((1 << 20, 1 << 20, 0),)),
                dict(buffers=((1 << 20, 1 << 20, 64), (1 << 20, 1 << 20, 0))),
                dict(buffers=((1 << 20, 1 << 20, 1 << 46),)),
                dict(buffers=((1 << 20, 1 << 20, (1 << 31) + 1),), slots=1),
                dict(buffers=((1 << 20, 1 << 20, 16),) * 64 + ((1 << 20, 1 << 20, 1 << 36),),
                     slots=1)):
        assert copy(**bad) == 1, bad


# ------------------------------------------- the functions, with a recorder for a library

@pytest.fixture
def calls(monkeypatch):
    seen = []

    def recorder(name):
        def launch(*args):
            seen.append((name, args))
            return 0
        return launch

    library = types.SimpleNamespace(**{name: recorder(name) for name in (
        "gated_delta_tree_launch_v1", "gated_delta_commit_launch_v1", "slot_moves_launch_v1",
        "compaction_moves_launch_v1", "copy_slots_launch_v1")})
    for module in (layer, slots):
        monkeypatch.setattr(module, "native", lambda: library)
        monkeypatch.setattr(module, "_stream", lambda: 0)
    monkeypatch.setattr(layer, "_current_device", lambda: torch.empty(0).get_device())
    return seen


def batch():
    q, k, v = (torch.zeros(10, n, 128).bfloat16() for n in (2, 2, 4))
    g, b = torch.zeros(10, 4), torch.zeros(10, 4).bfloat16()
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    tables = gdn.RequestTables(ints(3), ints(3), ints(2, 4), ints(2))
    return dict(queries=q, keys=k, values=v, log_decay=g, beta=b, parents=ints(10),
                tables=tables, slot_ids=ints(2), pool=torch.zeros(3, 4, 128, 128))


def test_what_trees_are_launched_with(calls):
    good = batch()
    out = gdn.gated_delta_tree(**good, max_nodes=5, scale=0.25, normalize=False)
    (name, args), = calls
    d = args[1]._obj
    assert name == "gated_delta_tree_launch_v1" and args[5] == out.data_ptr()
    assert (d.requests, d.tokens, d.value_heads, d.key_heads, d.max_nodes) == (2, 10, 4, 2, 5)
    assert (d.scale, d.normalize) == (0.25, 0)
    assert (d.query_stride, d.key_stride, d.value_stride) == (256, 256, 512)
    assert d.parents == good["parents"].data_ptr()
    good.pop("queries")
    accepted = torch.zeros(2, dtype=torch.int32)
    assert gdn.gated_delta_commit(**good, accepted=accepted) is None
    d = calls[1][1][1]._obj
    assert d.queries is None and d.max_nodes == 64 and calls[1][1][2] == accepted.data_ptr()


def test_trees_refuse_what_they_cannot_differentiate(calls):
    good = batch()
    for name in ("queries", "keys", "values", "log_decay", "beta", "pool"):
        with pytest.raises(RuntimeError, match="no gradient"):
            gdn.gated_delta_tree(**{**good, name: good[name].clone().requires_grad_()})
    with torch.no_grad():
        gdn.gated_delta_tree(**{**good, "values": good["values"].clone().requires_grad_()})
    assert len(calls) == 1


def test_what_copies_are_launched_with(calls):
    a, b = torch.zeros(6, 3, dtype=torch.int8), torch.zeros(6, 2, 5)
    moves = gdn.slot_moves(torch.zeros(4, dtype=torch.int32),
                           torch.zeros(4, dtype=torch.int32), 6)
    assert moves.slots == 6 and moves.steps.shape == (4, 4)
    gdn.copy_slots([a, b, torch.zeros(6, 0)], moves)
    args = calls[1][1]
    assert args[2:] == (2, moves.steps.data_ptr(), 4, 6)
    assert list(args[1]) == [a.data_ptr(), a.data_ptr(), 3, b.data_ptr(), b.data_ptr(), 40]
    into = torch.ones_like(b)
    gdn.copy_slots(b, moves, into=into)
    assert list(calls[2][1][1]) == [b.data_ptr(), into.data_ptr(), 40]
    gdn.copy_slots([b, b], moves, into=[into, torch.ones_like(b)])  # one source, two copies
    rows = torch.zeros(7, 4)  # what is only read may overlap
    gdn.copy_slots([rows[:6], rows[1:]], moves, into=[torch.ones(6, 4), torch.ones(6, 4)])
    for bad in (([b, b], moves), (b, moves, b), (b[:5], moves), ([], moves),
                ([b, b], moves, [into, into]), (b, moves, into[:, :1])):
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            gdn.copy_slots(*bad)


def test_compaction_tables(calls):
    for n in (1, 2, 7, 8):
        packed = gdn.compaction_moves(torch.zeros(n, dtype=torch.int32))
        assert packed.moves.slots == n and packed.moves.steps.shape == ((n + 1) // 2, 4)
        assert packed.placed.shape == (n,) and packed.count.shape == (1,)
        for t in (packed.moves.steps, packed.placed, packed.count):
            assert (t.data_ptr() - packed.moves.steps.data_ptr()) % 16 == 0
