"""gated_delta_commit's max_nodes: a node that the tree's call did not look at is not accepted."""

from __future__ import annotations

import pytest
import torch

import draft_reference as ref
import gdn_state_codec as gdn
from test_draft_tree_gpu import FP32, Batch, close, ints

pytestmark = pytest.mark.gpu


def _commit(batch, accepted, device, **more):
    gdn.gated_delta_commit(*batch.inputs()[1:], batch.dev_parents, ints(accepted, device),
                           batch.tables, batch.dev_slots, batch.dev_pool, **more)


@pytest.mark.parametrize("max_nodes", [1, 15, 16, 17, 32, 63, 64])
def test_nodes_past_the_limit_are_not_accepted(device, max_nodes):
    trees = [ref.parents_of("chain", n) for n in (64, 64, 70, 20, 3)]
    batch = Batch(device, trees, 4, 2, torch.float32, 91, padded=False)
    accepted = [max_nodes - 1, max_nodes, 69, 19, 2]
    _commit(batch, accepted, device, max_nodes=max_nodes)
    for r, tree in enumerate(trees):
        got = batch.dev_pool[int(batch.slots[r])]
        if accepted[r] < min(max_nodes, len(tree)):
            close(got, batch.reference(r)[1][accepted[r]], FP32, f"state {r}")
        else:
            assert torch.equal(got.cpu(), batch.pool[int(batch.slots[r])])


def test_refusals(device):
    batch = Batch(device, [ref.parents_of("chain", 4)], 2, 1, torch.float32, 93)
    for bad in (0, 65, -1):
        with pytest.raises(RuntimeError, match="max_nodes"):
            _commit(batch, [3], device, max_nodes=bad)
    assert torch.equal(batch.dev_pool.cpu(), batch.pool)
