"""Training through the layer operators as programs run it: checkpointed, offloaded and
captured, against the plain call.  The kernels give the same bits for the same inputs
(no atomics), so the gradients are equal, not close."""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import gdn_state_codec as gdn

pytestmark = pytest.mark.gpu

LENGTHS, HEADS, KEY_HEADS = [130, 0, 64, 7], 4, 2


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.fixture
def batch(device):
    """Leaves (one fused projection, decays, strengths, states, gate, weight), tables and
    the gradients of the output and the final states."""
    gen = torch.Generator().manual_seed(71)
    total = sum(LENGTHS)

    def made(*shape):
        return torch.randn(shape, generator=gen).to(device)

    leaves = [made(total, (2 * KEY_HEADS + HEADS) * 128).bfloat16(),
              -0.2 * made(total, HEADS).abs(), torch.sigmoid(made(total, HEADS)).bfloat16(),
              0.1 * made(len(LENGTHS), HEADS, 128, 128), made(total, HEADS, 128).bfloat16(),
              1.0 + 0.1 * made(128)]
    tables = gdn.request_tables(ints(LENGTHS, device), ints(range(len(LENGTHS)), device), total)
    given = [made(total, HEADS, 128).bfloat16(), made(len(LENGTHS), HEADS, 128, 128)]
    return [x.requires_grad_() for x in leaves], tables, given


def block(mixed, log_decay, beta, initial, gate, weight, tables):
    q, k, v = (x.unflatten(1, (-1, 128)) for x in
               mixed.split((KEY_HEADS * 128, KEY_HEADS * 128, HEADS * 128), 1))
    out, final = gdn.gated_delta_rule(q, k, v, log_decay, beta, tables, initial)
    normed = gdn.gated_norm(out, gate, weight)
    stream = torch.zeros(normed.shape, device=normed.device)
    return gdn.residual_norm(normed, stream, weight)[0], final


def gradients(outs, leaves, given):
    """The gradients, with the caching allocator's free blocks taken and watched."""
    others = [torch.full((1 << 20,), 5.0, device=given[0].device) for _ in range(24)]
    got = torch.autograd.grad(outs, leaves, given)
    assert all(bool((x == 5.0).all()) for x in others)
    return got


def test_checkpointed(batch):
    leaves, tables, given = batch
    want = gradients(block(*leaves, tables), leaves, given)
    got = gradients(checkpoint(block, *leaves, tables, use_reentrant=False), leaves, given)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_checkpointed_blocks(batch):
    leaves, tables, given = batch

    def both(run):
        first, state = run(*leaves, tables)
        return run(*leaves[:3], state, first, leaves[5], tables)

    want = gradients(both(block), leaves, given)
    got = gradients(both(lambda *x: checkpoint(block, *x, use_reentrant=False)), leaves, given)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("hooks", [
    lambda: torch.autograd.graph.save_on_cpu(),
    lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t)])
def test_saved_elsewhere(batch, hooks):
    leaves, tables, given = batch
    want = gradients(block(*leaves, tables), leaves, given)
    with hooks():
        outs = block(*leaves, tables)
    for a, b in zip(gradients(outs, leaves, given), want):
        assert torch.equal(a, b)


def test_gradients_that_start_anywhere(batch):
    """Outputs joined behind an odd number of values: their gradients are unaligned slices."""
    leaves, tables, given = batch
    want = gradients(block(*leaves, tables), leaves, given)
    outs = block(*leaves, tables)
    joined = torch.cat([given[1].new_zeros(3)] + [x.float().flatten() for x in outs])
    d = torch.cat([given[1].new_zeros(3)] + [x.float().flatten() for x in given])
    for a, b in zip(gradients([joined], leaves, [d]), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("lengths", [[130, 0, 64, 7], [130, 0, 64, 7] * 3])
def test_a_captured_training_pass_replays(device, lengths):
    gen = torch.Generator().manual_seed(73)
    total = sum(lengths)

    def made(*shape):
        return torch.randn(shape, generator=gen).to(device)

    leaves = [made(total, (2 * KEY_HEADS + HEADS) * 128).bfloat16(),
              -0.2 * made(total, HEADS).abs(), torch.sigmoid(made(total, HEADS)).bfloat16(),
              0.1 * made(len(lengths), HEADS, 128, 128), made(total, HEADS, 128).bfloat16(),
              1.0 + 0.1 * made(128)]
    leaves = [x.requires_grad_() for x in leaves]
    given = [made(total, HEADS, 128).bfloat16(), made(len(lengths), HEADS, 128, 128)]
    lens, slots = ints(lengths, device), ints(range(len(lengths)), device)

    def work():
        tables = gdn.request_tables(lens, slots, total)
        outs = block(*leaves, tables)
        return [*(x.detach() for x in outs), *torch.autograd.grad(outs, leaves, given)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for i in range(3):
        with torch.no_grad():
            leaves[0].mul_(0.5 + 0.25 * i)
        eager = [x.clone() for x in work()]
        for x in held:
            x.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b)
