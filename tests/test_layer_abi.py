"""The layer operators' C-ABI on a machine without a GPU: bad arguments return 1
before any HIP call, and sizes are what the header says."""

from __future__ import annotations

import ctypes

import pytest

from gdn_state_codec import _native
from gdn_state_codec._native import RuleStruct

P = ctypes.c_void_p(1 << 20)  # 16-byte aligned, never dereferenced


@pytest.fixture(scope="module")
def lib():
    return _native.NativeLibrary()


def _each_pointer(call, count, optional=(), by_element=()):
    """call(*pointers) is refused with any one of its pointers null or misaligned
    (to 16 bytes, or to an element)."""
    for i in range(count):
        args = [P] * count
        args[i] = None
        if i not in optional:
            assert call(*args) == 1, i
        args[i] = ctypes.c_void_p((1 << 20) + (1 if i in by_element else 4))
        assert call(*args) == 1, i


def test_request_tables_admission(lib):
    def call(*p, n=4, tokens=100, rows=5):
        return lib.request_tables_launch_v1(None, p[0], p[1], n, tokens, rows, *p[2:])

    _each_pointer(call, 6)
    assert call(*[P] * 6, n=0, rows=1) == 1
    assert call(*[P] * 6, n=4097, rows=4098) == 1
    assert call(*[P] * 6, rows=6) == 1
    assert call(*[P] * 6, tokens=1 << 31, rows=(1 << 25) + 4) == 1


def test_gated_delta_step_admission(lib):
    def call(*p, batch=2, slots=3, heads=4, key_heads=2, strides=(256, 256, 512), dtype=0,
             normalize=1):
        return lib.gated_delta_step_launch_v1(None, *p, batch, slots, heads, key_heads, *strides,
                                              dtype, 1.0, normalize)

    _each_pointer(call, 8, by_element=(3, 4))
    for bad in (dict(batch=0), dict(slots=0), dict(heads=0), dict(key_heads=0),
                dict(heads=3), dict(strides=(4, 256, 512)), dict(strides=(256, 260, 512)),
                dict(strides=(256, 256, 513)), dict(dtype=2), dict(normalize=2),
                dict(slots=1 << 31)):
        assert call(*[P] * 8, **bad) == 1, bad


POINTERS = ("queries", "keys", "values", "log_decay", "beta", "offsets", "chunk_offsets",
            "chunks", "order", "workspace")


def _rule(lib, train, **changes):
    fields = {name: P for name in POINTERS}
    fields.update(query_stride=256, key_stride=256, value_stride=512, requests=3, rows=7,
                  tokens=300, value_heads=4, key_heads=2, scale=1.0, normalize=1)
    fields.update(changes)
    if "workspace_bytes" not in fields:
        fields["workspace_bytes"] = lib.gated_delta_workspace_v1(
            fields["rows"], fields["value_heads"], fields["key_heads"], train)
    return RuleStruct(**fields)


@pytest.mark.parametrize("entry", ["prefill", "forward", "backward"])
def test_whole_sequence_admission(lib, entry):
    train = entry != "prefill"

    def call(rule):
        r = None if rule is None else ctypes.byref(rule)
        if entry == "prefill":
            return lib.gated_delta_prefill_launch_v1(None, r, P, None, P, 4, 0, P)
        if entry == "forward":
            return lib.gated_delta_forward_launch_v1(None, r, None, P, P)
        return lib.gated_delta_backward_launch_v1(None, r, P, None, P, P, P, P, P, None)

    assert call(None) == 1
    for name in POINTERS:
        assert call(_rule(lib, train, **{name: None})) == 1, name
        off = 1 if name in ("log_decay", "beta") else 8
        assert call(_rule(lib, train, **{name: ctypes.c_void_p((1 << 20) + off)})) == 1, name
    enough = _rule(lib, train).workspace_bytes
    for bad in (dict(requests=0, rows=4), dict(requests=4097, rows=4101), dict(rows=8),
                dict(value_heads=3), dict(key_heads=0), dict(value_heads=0), dict(normalize=2),
                dict(query_stride=252), dict(key_stride=(1 << 24) + 8), dict(value_stride=513),
                dict(workspace_bytes=enough - 1), dict(tokens=1 << 31, rows=(1 << 25) + 3)):
        assert call(_rule(lib, train, **bad)) == 1, bad


def test_prefill_state_arguments(lib):
    rule = _rule(lib, False)

    def call(slot_ids=P, resume=None, pool=P, slots=4, dtype=0, outputs=P):
        return lib.gated_delta_prefill_launch_v1(None, ctypes.byref(rule), slot_ids, resume, pool,
                                                 slots, dtype, outputs)

    off = ctypes.c_void_p((1 << 20) + 4)
    for bad in (dict(slot_ids=None), dict(pool=None), dict(outputs=None), dict(slots=0),
                dict(dtype=2), dict(slot_ids=off), dict(resume=off), dict(pool=off),
                dict(outputs=off), dict(slots=1 << 31)):
        assert call(**bad) == 1, bad


def test_norm_admission(lib):
    def gated(*p, rows=4, dtype=0):
        return lib.gated_norm_launch_v1(None, *p, rows, dtype, 1e-6)

    def gated_back(*p, rows=4, dtype=0):
        return lib.gated_norm_backward_launch_v1(None, *p, rows, dtype, 1e-6)

    def residual(*p, rows=4, width=64, dtype=0, stream=0):
        return lib.residual_norm_launch_v1(None, *p, rows, width, dtype, stream, 1.0, 1e-6)

    def residual_back(*p, rows=4, width=64, dtype=0, stream=0):
        return lib.residual_norm_backward_launch_v1(None, *p, rows, width, dtype, stream, 1.0,
                                                    1e-6)

    _each_pointer(gated, 4)
    _each_pointer(gated_back, 8)
    _each_pointer(residual, 5)
    _each_pointer(residual_back, 8, optional=(3,))
    for call, n in ((gated, 4), (gated_back, 8), (residual, 5), (residual_back, 8)):
        assert call(*[P] * n, rows=0) == 1
        assert call(*[P] * n, dtype=2) == 1
    for call, n in ((residual, 5), (residual_back, 8)):
        for bad in (dict(width=0), dict(width=12), dict(width=16392), dict(stream=2)):
            assert call(*[P] * n, **bad) == 1, bad


def test_sizes(lib):
    assert lib.norm_partials_v1(1, 128) == 1
    assert lib.norm_partials_v1(5, 128) == 2
    assert lib.norm_partials_v1(1 << 20, 128) == 1024
    assert lib.norm_partials_v1(1 << 20, 4096) == 512
    one, two = (lib.gated_delta_workspace_v1(n, 4, 2, 0) for n in (1, 2))
    assert 0 < one < two < 2 * one
    # Training keeps each chunk's start state and its gradient (64 KiB a head) too.
    assert lib.gated_delta_workspace_v1(1, 4, 2, 1) - one > 4 * 2 * 65536


def test_workspace_holds_the_states_between_segments(lib):
    """256 states of 64 KiB from 64 chunk rows on, for up to 32 heads, serving only."""
    def step(rows, heads, train):
        size = lib.gated_delta_workspace_v1
        return size(rows, heads, 1, train) - size(rows - 1, heads, 1, train)

    states = 256 * 65536
    assert step(64, 32, 0) == step(63, 32, 0) + states
    assert step(64, 33, 0) == step(63, 33, 0)
    assert step(64, 32, 1) == step(63, 32, 1)
