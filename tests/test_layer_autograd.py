"""The layer operators' autograd functions on a machine without a GPU: the native
library is replaced by a recorder that launches nothing, and what it is called with is
held to the tensors that are alive at that call."""

from __future__ import annotations

import types

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import gdn_state_codec as gdn
from gdn_state_codec import _native, layer
from gdn_state_codec._native import RuleStruct

HEADS, KEY_HEADS, TOKENS = 4, 2, 70
POINTERS = ("queries", "keys", "values", "log_decay", "beta", "offsets", "chunk_offsets",
            "chunks", "order", "workspace")


@pytest.fixture
def calls(monkeypatch):
    """(name, arguments) of every launch; a rule's struct as a dict of its fields."""
    seen = []
    real = _native.NativeLibrary()

    def recorder(name):
        def launch(*args):
            args = [{field: getattr(a._obj, field) for field, _ in RuleStruct._fields_}
                    if hasattr(a, "_obj") else a for a in args]
            seen.append((name, args))
            return 0
        return launch

    library = types.SimpleNamespace(
        gated_delta_workspace_v1=real.gated_delta_workspace_v1,
        norm_partials_v1=real.norm_partials_v1,
        **{name: recorder(name) for name in (
            "gated_delta_forward_launch_v1", "gated_delta_backward_launch_v1",
            "gated_delta_prefill_launch_v1", "gated_delta_step_launch_v1",
            "gated_norm_launch_v1", "gated_norm_backward_launch_v1",
            "residual_norm_launch_v1", "residual_norm_backward_launch_v1")})
    monkeypatch.setattr(layer, "native", lambda: library)
    monkeypatch.setattr(layer, "_stream", lambda: 0)
    monkeypatch.setattr(layer, "_current_device", lambda: torch.empty(0).get_device())
    return seen


def batch(tokens=TOKENS, requests=2):
    """Leaves (queries, keys and values slices of one projection) and tables."""
    mixed = torch.randn(tokens, (2 * KEY_HEADS + HEADS) * 128).bfloat16()
    q, k, v = (x.unflatten(1, (-1, 128)) for x in
               mixed.split((KEY_HEADS * 128, KEY_HEADS * 128, HEADS * 128), 1))
    rest = [torch.zeros(tokens, HEADS), torch.zeros(tokens, HEADS).bfloat16()]
    rows = layer.table_rows(tokens, requests)
    tables = gdn.RequestTables(*(torch.zeros(shape, dtype=torch.int32) for shape in (
        requests + 1, requests + 1, (rows, 4), requests)))
    return [x.detach().requires_grad_() for x in (q, k, v, *rest)], tables


def struct_of(tensors):
    """The pointers and strides that a rule's saved tensors ask for."""
    want = dict(zip(POINTERS, (t.data_ptr() for t in tensors)))
    want.update(zip(("query_stride", "key_stride", "value_stride"),
                    (t.stride(0) for t in tensors)))
    want["workspace_bytes"] = tensors[9].numel()
    return want


def check(rule, tensors):
    want = struct_of(tensors)
    assert {name: rule[name] for name in want} == want


def test_backward_reads_what_the_saved_tensors_were_unpacked_to(calls):
    leaves, tables = batch()
    unpacked = []

    def unpack(t):
        unpacked.append(t)
        return t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
        out, final = gdn.gated_delta_rule(*leaves, tables)
    torch.autograd.grad([out], leaves, [torch.ones_like(out)])
    (_, forward), (name, backward) = calls
    assert name == "gated_delta_backward_launch_v1" and len(unpacked) == 10
    check(backward[1], unpacked)
    assert unpacked[0].stride(0) == KEY_HEADS * 128  # a copy of the slice is dense
    for field in ("requests", "rows", "tokens", "value_heads", "key_heads", "scale", "normalize"):
        assert backward[1][field] == forward[1][field]


def test_backward_reads_what_a_checkpoint_recomputed(calls):
    leaves, tables = batch()
    kept = []  # of every forward call, so that no address is used twice

    def block(*inputs):
        inputs = [x * 1.0 for x in inputs]
        out, final = gdn.gated_delta_rule(*inputs, tables)
        kept.append(inputs + [out, final])
        return out, final

    out, final = checkpoint(block, *leaves, use_reentrant=False)
    torch.autograd.grad([out, final], leaves, [torch.ones_like(out), torch.ones_like(final)])
    names = [name.split("_")[2] for name, _ in calls]
    assert names == ["forward", "forward", "backward"]
    for field in POINTERS:
        assert calls[2][1][1][field] == calls[1][1][1][field], field


def test_backward_without_hooks_reads_the_forward_call_s_tensors(calls):
    leaves, tables = batch()
    out, final = gdn.gated_delta_rule(*leaves, tables)
    torch.autograd.grad([out], leaves, [torch.ones_like(out)])
    assert calls[0][1][1] == calls[1][1][1]


def test_backward_refuses_what_a_hook_changed(calls):
    leaves, tables = batch()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:-1]):
        out, _ = gdn.gated_delta_rule(*leaves, tables)
    with pytest.raises(RuntimeError, match="GDN State Codec"):
        torch.autograd.grad([out], leaves, [torch.ones_like(out)])
    assert len(calls) == 1


@pytest.mark.parametrize("operator", ["rule", "gated norm", "residual norm"])
def test_gradients_that_start_anywhere(calls, operator):
    """The gradient of a torch.cat's operand is a slice of the whole one, and starts where
    the operand did: no 16-byte boundary."""
    if operator == "rule":
        leaves, tables = batch()
        outs = gdn.gated_delta_rule(*leaves, tables)
    elif operator == "gated norm":
        leaves = [torch.randn(3, 128).requires_grad_() for _ in range(2)]
        leaves.append(torch.ones(128).requires_grad_())
        outs = (gdn.gated_norm(*leaves),)
    else:
        leaves = [torch.randn(3, 64).requires_grad_() for _ in range(2)]
        leaves.append(torch.ones(64).requires_grad_())
        outs = gdn.residual_norm(*leaves)
    joined = torch.cat([torch.zeros(3)] + [x.float().flatten() for x in outs])
    torch.autograd.grad([joined], leaves, [torch.randn_like(joined)])
    name, args = calls[-1]
    assert "backward" in name
    pointers = args[2:] if operator == "rule" else args[1:9]
    assert len(pointers) == 8
    for pointer in pointers:
        assert pointer % 16 == 0


def norm_inputs():
    return {gdn.gated_norm: [torch.randn(3, 128), torch.randn(3, 128), torch.ones(128)],
            gdn.residual_norm: [torch.randn(3, 64), torch.randn(3, 64), torch.ones(64)]}


@pytest.mark.parametrize("norm", [gdn.gated_norm, gdn.residual_norm])
@pytest.mark.parametrize("place", range(3))
def test_norms_refuse_tangents(calls, norm, place):
    """There is no forward-mode derivative: a dual tensor is refused, not cut off."""
    inputs = norm_inputs()[norm]
    with torch.autograd.forward_ad.dual_level():
        norm(*inputs)  # no dual among them
        inputs[place] = torch.autograd.forward_ad.make_dual(inputs[place],
                                                            torch.ones_like(inputs[place]))
        launched = len(calls)
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            norm(*inputs)
    assert len(calls) == launched == 1

def serving_calls():
    """The two calls that update a pool in place, as functions of their float inputs."""
    leaves, tables = batch()
    inputs = [x.detach() for x in leaves]
    slots = torch.zeros(TOKENS, dtype=torch.int32)
    inputs.append(torch.zeros(3, HEADS, 128, 128))
    return inputs, {
        "step": lambda *x: gdn.gated_delta_step(*x, slots),
        "prefill": lambda *x: gdn.gated_delta_prefill(*x[:5], tables, slots[:2], x[5])}


@pytest.mark.parametrize("call", ["step", "prefill"])
@pytest.mark.parametrize("place", range(6))
def test_serving_calls_refuse_what_they_cannot_differentiate(calls, call, place):
    """Inputs and states of a serving call that require gradients, or hold tangents."""
    inputs, functions = serving_calls()
    functions[call](*inputs)
    wanted = list(inputs)
    wanted[place] = inputs[place].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="GDN State Codec"):
        functions[call](*wanted)
    with torch.autograd.forward_ad.dual_level():
        functions[call](*inputs)
        dual = list(inputs)
        dual[place] = torch.autograd.forward_ad.make_dual(
            inputs[place].clone(), torch.ones_like(inputs[place]))
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            functions[call](*dual)
    assert len(calls) == 2
    with torch.no_grad():
        functions[call](*wanted)
    assert len(calls) == 3


@pytest.mark.parametrize("place,shape", [(0, ()), (0, (TOKENS,)), (1, ()), (1, (TOKENS,)),
                                         (2, ()), (2, (TOKENS,)), (3, ()), (4, ())])
def test_inputs_without_dimensions_are_refused(calls, place, shape):
    leaves, tables = batch()
    inputs = [x.detach() for x in leaves]
    inputs[place] = torch.zeros(shape, dtype=inputs[place].dtype)
    pool = torch.zeros(3, HEADS, 128, 128)
    slots = torch.zeros(TOKENS, dtype=torch.int32)
    for call in (lambda: gdn.gated_delta_step(*inputs, pool, slots),
                 lambda: gdn.gated_delta_prefill(*inputs, tables, slots[:2], pool),
                 lambda: gdn.gated_delta_rule(*inputs, tables),
                 lambda: gdn.gated_delta_rule(*inputs, tables, pool[:2])):
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            call()
    assert not calls
