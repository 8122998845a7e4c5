"""Trees of drafted tokens and moves between slots straight from their definitions, on the
CPU and in float64: what the kernels of ``gdn_state_codec.layer`` and ``slots`` are held to."""

from __future__ import annotations

import random

import torch

from delta_reference import DIM, expanded


def parents_of(shape: str, nodes: int, seed: int = 0) -> list[int]:
    """Each node's parent: a chain, a star below node 0, two branches, all roots, or any
    earlier node (or the cached state)."""
    rng = random.Random(1000 * seed + nodes)
    if shape == "chain":
        return list(range(-1, nodes - 1))
    if shape == "star":
        return [-1] + [0] * (nodes - 1) if nodes else []
    if shape == "branches":
        return [-1] + [max(0, i - 2) for i in range(1, nodes)] if nodes else []
    if shape == "roots":
        return [-1] * nodes
    return [rng.randint(-1, i - 1) for i in range(nodes)]


def path(parents: list[int], node: int) -> list[int]:
    """The nodes from the cached state down to `node`."""
    found = []
    while node >= 0:
        found.append(node)
        above = parents[node]
        node = above if 0 <= above < node else -1
    return found[::-1]


def tree(queries, keys, values, log_decay, beta, parents, initial, scale=DIM ** -0.5,
         normalize=True):
    """out [T,H,128] and every node's state [T,H,128 value,128 key] of one request's tree
    (float64), from initial [H,128 value,128 key]: S = a S_parent; e = v - S k;
    S <- S + b e k^T; o = S q."""
    heads = values.shape[1]
    q, k = expanded(queries, keys, heads // keys.shape[1], scale, normalize)
    v, a, b = values.double(), log_decay.double().exp(), beta.double()
    nodes = len(parents)
    out = torch.zeros((nodes, heads, DIM), dtype=torch.float64)
    states = torch.zeros((nodes, heads, DIM, DIM), dtype=torch.float64)
    for i, above in enumerate(parents):
        state = states[above] if 0 <= above < i else initial.double()
        state = state * a[i][:, None, None]
        error = v[i] - torch.matmul(state, k[i][:, :, None])[..., 0]
        states[i] = state + (b[i][:, None] * error)[:, :, None] * k[i][:, None, :]
        out[i] = torch.matmul(states[i], q[i][:, :, None])[..., 0]
    return out, states


def moved(rows: torch.Tensor, sources, targets) -> torch.Tensor:
    """Every target with what its source held before; -1 clears, pairs outside are left
    out, the last pair of a target counts."""
    after, slots = rows.clone(), rows.shape[0]
    for source, target in zip(sources, targets):
        if 0 <= target < slots and -1 <= source < slots:
            after[target] = rows[source] if source >= 0 else 0
    return after


def compacted(live) -> tuple:
    """(sources, targets, placed, count) of packing live slots to the front."""
    count = sum(1 for x in live if x)
    free = [i for i in range(count) if not live[i]]
    late = [i for i in range(count, len(live)) if live[i]]
    to = dict(zip(late, free))
    return late, free, [to.get(i, i) if x else -1 for i, x in enumerate(live)], count
