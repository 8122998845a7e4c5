"""Trees of drafted tokens whose writes pass fp32's range on one branch, from inputs that are
all finite (gated_delta_tree, gated_delta_commit): no other branch's outputs change, and what
is finite by the definition is as good as ever."""

from __future__ import annotations

import pytest
import torch

import draft_reference as ref
from test_draft_tree_gpu import BF16, FP32, Batch, close

pytestmark = pytest.mark.gpu


def _others(nodes, apart, seed):
    """Parents of `nodes` nodes, none of them one of `apart`."""
    parents = ref.parents_of("any", nodes, seed)
    return [-1 if p in apart else p for p in parents]


@pytest.mark.parametrize("first,second", [
    (3.0e38, -3.0e38),            # the child's write is -6e38
    (1.0e36, -float.fromhex("0x1.fep127")),  # and here past the largest bf16 alone
])
@pytest.mark.parametrize("node,nodes", [(1, 14), (1, 40), (9, 30), (20, 30), (20, 64), (40, 64)])
@pytest.mark.parametrize("pool_dtype", [torch.float32, torch.bfloat16])
def test_a_write_that_overflows_stays_on_its_branch(device, pool_dtype, node, nodes, first,
                                                    second):
    """Node 0 and its child `node` write opposite values to one key, all of them finite; their
    sum is not.  Every other node's outputs are the very same as with small values there,
    before and after it, in its tile of 16 and in others."""
    parents = _others(nodes, (0, node, nodes - 1), 21)
    parents[0], parents[node], parents[nodes - 1] = -1, 0, node
    batch = Batch(device, [parents, ref.parents_of("any", 20, 22)], 4, 2, pool_dtype, 61,
                  padded=False, rest=0)
    batch.mixed[node, 256:384] = batch.mixed[0, 256:384]  # the key of heads 0 and 1
    batch.g[[0, node]], batch.b[[0, node]] = 0.0, 1.0
    column = 512 + 128 + 77  # head 1's
    batch.mixed[0, column], batch.mixed[node, column] = 1.0, -1.0
    for dev, cpu in ((batch.dev_mixed, batch.mixed), (batch.dev_g, batch.g),
                     (batch.dev_b, batch.b)):
        dev.copy_(cpu)
    clean = batch.tree().cpu()
    batch.dev_mixed[0, column], batch.dev_mixed[node, column] = first, second
    got = batch.tree().cpu()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[[0, node, nodes - 1], 1, 77] = True
    assert torch.equal(got[~hit], clean[~hit])
    assert torch.isfinite(got[0]).all()
    if first == 3.0e38:
        assert not torch.isfinite(got[node, 1, 77])


def _steep(device, nodes, chain, pool_dtype, last=None):
    """A chain at the places `chain` over one long key, so that each node's write is some
    10,000 times the one above it, among short branches of ordinary ones; the cached state is
    zeros, and so are the chain's values but those of place `last`, where that is given."""
    parents = _others(nodes, chain, 23)
    for above, node in zip([-1] + chain, chain):
        parents[node] = above
    batch = Batch(device, [parents], 2, 1, pool_dtype, 67, normalize=False, decay="none",
                  padded=False, rest=0)
    key = batch.mixed[0, 128:256].float()
    batch.mixed[chain, 128:256] = (100.0 / key.norm() * key).bfloat16()
    batch.b[chain] = 1.0
    if last is not None:
        batch.mixed[chain, 256:] = 0.0
        batch.mixed[last, 256:] = 1.0
        batch.pool.zero_()
    batch.dev_mixed.copy_(batch.mixed)
    batch.dev_b.copy_(batch.b)
    batch.dev_pool.copy_(batch.pool)
    return batch


@pytest.mark.parametrize("pool_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nodes,chain", [
    (16, list(range(0, 16, 2)) + [13, 15]), (16, list(range(14))),
    (30, list(range(1, 30, 2))), (64, list(range(0, 24))), (64, list(range(3, 60, 4)))])
def test_keys_that_grow_a_branch_past_the_range(device, nodes, chain, pool_dtype):
    """Every output that is finite by the definition, with its states and writes in fp32's
    range, is held to it, and what is not in range has no finite value.  (Ranges: an output
    is a state's row times a query of some 6, so that 1e36 leaves it and the states above it
    in range, and 1e41 does not.)"""
    chain = sorted(set(chain))
    batch = _steep(device, nodes, chain, pool_dtype)
    got = batch.tree().cpu()
    want, states = batch.reference(0)
    largest = states.abs().flatten(1).amax(1)
    for node in range(nodes):
        above = max(largest[i] for i in ref.path(batch.parents[0], node))
        if above < 1e36:
            for head in range(2):
                close(got[node, head], want[node, head], 2.0 ** -7, f"node {node}")
        elif above > 1e41:
            assert not torch.isfinite(got[node]).any(), node


@pytest.mark.parametrize("pool_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nodes,places,last", [
    (14, range(0, 14), 10), (30, range(16, 30), 27), (64, range(32, 48), 44),
    (64, range(0, 64, 3), 60)])
def test_growth_that_no_write_meets(device, nodes, places, last, pool_dtype):
    """A chain's factors from its first node to its last pass fp32's range by far, but the
    nodes before its last few write nothing: all is finite, states too."""
    chain = list(places)
    batch = _steep(device, nodes, chain, pool_dtype, last)
    got = batch.tree().cpu()
    want, states = batch.reference(0)
    for node in range(nodes):
        for head in range(2):
            close(got[node, head], want[node, head], 2.0 ** -7, f"node {node}")
    batch.commit([chain[-1]])
    exact = pool_dtype == torch.float32
    close(batch.dev_pool[int(batch.slots[0])], states[chain[-1]], FP32 if exact else BF16,
          "state")


@pytest.mark.parametrize("pool_dtype", [torch.float32, torch.bfloat16])
def test_growth_with_decays(device, pool_dtype):
    """The same on a path with decays, one of them -inf before the writes."""
    chain = list(range(20))
    batch = _steep(device, 20, chain, pool_dtype, 16)
    batch.g.uniform_(-0.5, 0.0, generator=torch.Generator().manual_seed(69))
    batch.g[2] = float("-inf")
    batch.pool.normal_(generator=torch.Generator().manual_seed(70)).mul_(1e-30)
    batch.dev_g.copy_(batch.g)
    batch.dev_pool.copy_(batch.pool)
    want, states = batch.reference(0)
    got = batch.tree().cpu()
    for node in range(3, 20):
        for head in range(2):
            close(got[node, head], want[node, head], 2.0 ** -7, f"node {node}")
    batch.commit([19])
    close(batch.dev_pool[int(batch.slots[0])], states[19],
          FP32 if pool_dtype == torch.float32 else BF16, "state")


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("what", ["value", "strength", "key"])
@pytest.mark.parametrize("nodes,chain", [(16, range(0, 14)), (64, range(16, 31))])
def test_bad_values_beside_steep_keys(device, nodes, chain, what, bad):
    """A bad node beside a chain whose inverse is past the range: neither reaches the other."""
    chain = list(chain)
    batch = _steep(device, nodes, chain, torch.float32, chain[-3])
    node = chain[-1] + 1
    want, _ = batch.reference(0)
    if what == "value":
        batch.dev_mixed[node, 256 + 128 + 9] = bad  # head 1's column 9
    elif what == "strength":
        batch.dev_b[node, 1] = bad
    else:
        batch.dev_mixed[node, 128 + 3] = bad
    got = batch.tree().cpu()
    for i in range(nodes):
        reached = node in ref.path(batch.parents[0], i)
        for head in range(2):
            if not reached or (what != "key" and head == 0):
                close(got[i, head], want[i, head], 2.0 ** -7, f"node {i}")
            else:
                columns = [9] if what == "value" else range(128)
                assert not torch.isfinite(got[i, head, list(columns)]).any()
