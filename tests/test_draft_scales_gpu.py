"""Trees of drafted tokens whose heads and nodes differ in size by many powers of ten
(gated_delta_tree, gated_delta_commit): every cell is held to its own bound
(tests/draft_bounds.py), so that the largest head's error hides no other's."""

from __future__ import annotations

import types

import pytest
import torch

import draft_bounds as bounds
import draft_reference as ref
import gdn_state_codec as gdn
from test_draft_tree_gpu import Batch

TREES = (("chain", 64), ("any", 50), ("branches", 33), ("chain", 17), ("roots", 20))
HALF_STEP = 2.0 ** -8  # of bf16


def batch_of(device, kind, pool_dtype):
    shapes = [ref.parents_of(s, n, 31) for s, n in TREES]
    normalize = kind != "unnormalized"
    batch = Batch(device, shapes, 4, 2, pool_dtype, 83, normalize,
                  "strong" if kind == "strong" else "mixed", padded=False)
    if kind == "growing":  # by up to e^32
        batch.g.uniform_(-0.3, 0.5, generator=torch.Generator().manual_seed(83))
        batch.g[:64, 0] = 0.5
        batch.dev_g.copy_(batch.g)
    return batch


def arguments(batch, r):
    at = slice(batch.starts[r], batch.starts[r] + len(batch.parents[r]))
    mixed = batch.mixed[at]
    q, k, v = (mixed[:, :256].view(-1, 2, 128), mixed[:, 256:512].view(-1, 2, 128),
               mixed[:, 512:].view(-1, 4, 128))
    return (q, k, v, batch.g[at], batch.b[at], batch.parents[r],
            batch.pool[int(batch.slots[r])], batch.scale, batch.normalize)


KINDS = ("growing", "strong", "unnormalized", "mixed")


@pytest.mark.parametrize("kind", KINDS)
def test_the_bounds_say_something(monkeypatch, kind):
    """Every output vector and every state is many times its bound."""
    monkeypatch.setattr(gdn, "request_tables", lambda *_: types.SimpleNamespace())
    batch = batch_of(torch.device("cpu"), kind, torch.float32)
    shares = []
    for r, parents in enumerate(batch.parents):
        out, states = batch.reference(r)
        shares.append((bounds.outputs(*arguments(batch, r)).norm(dim=-1)
                       / out.norm(dim=-1)).flatten())
        off = bounds.state(*arguments(batch, r), len(parents) - 1)
        share = (off.flatten(1).norm(dim=1) / states[-1].flatten(1).norm(dim=1)).max()
        print(f"state {float(share):.3g}")
        assert share < 2.0 ** -5
    shares = torch.cat(shares)
    print(f"outputs {float(shares.median()):.3g}, worst {float(shares.max()):.3g}")
    assert shares.median() < 2.0 ** -10 and shares.max() < 2.0 ** -5


def _within(got, want, bound, name):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), name
    worst = float(((got - want).abs() / (bound + 1e-30)).max())
    print(f"{name}: {worst:.3g}", flush=True)
    assert worst <= 1.0, name


@pytest.mark.gpu
@pytest.mark.parametrize("pool_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
def test_every_cell_is_within_its_bound(device, kind, pool_dtype):
    batch = batch_of(device, kind, pool_dtype)
    out = batch.tree()
    batch.commit([len(p) - 1 for p in batch.parents])
    for r, parents in enumerate(batch.parents):
        want, states = batch.reference(r)
        at = batch.starts[r]
        bound = bounds.outputs(*arguments(batch, r))
        _within(out[at:at + len(parents)], want,
                bound + HALF_STEP * (want.abs() + bound), f"outputs {r}")
        bound = bounds.state(*arguments(batch, r), len(parents) - 1)
        if pool_dtype == torch.bfloat16:
            bound = bound + HALF_STEP * (states[-1].abs() + bound)
        _within(batch.dev_pool[int(batch.slots[r])], states[-1], bound, f"state {r}")
