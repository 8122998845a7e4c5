"""How far the outputs and states of a drafted tree may be from float64, cell by cell, from the
arithmetic: each term of each sum of fp32 numbers is off by EPS of its size, and what is off
goes on into what is formed from it (first order).

EPS = 2^-18 is 64 roundings of 2^-24.  A product with a state or of two keys sums 128 exact
products (three parts each of a state) in 12 instructions of 32 at a time, some 20 roundings;
a factor exp(G_i - G_j) is off by 2^-24 of its exponent (32 at most here: 2^-19) and an ulp or
two of the exponential, and has four products and a reciprocal root beside it."""

from __future__ import annotations

import torch

import draft_reference as ref
from delta_reference import expanded

EPS = 2.0 ** -18


def _writes(q, k, v, g, b, parents, initial, off):
    """Of one head: each node's decay from the state and from the nodes above it, and the
    writes' sizes and how far they may be off [nodes,128], from a state that is off by `off`."""
    n = len(parents)
    above = torch.zeros((n, n), dtype=torch.float64)
    for t in range(n):
        above[t, ref.path(parents, t)] = 1.0
    total = above @ g
    decay = torch.where(above > 0, torch.exp(total[:, None] - total[None, :]), 0.0)
    strict = decay * (1.0 - torch.eye(n, dtype=torch.float64)) * b[:, None]
    inverse = torch.linalg.inv(torch.eye(n, dtype=torch.float64) + strict * (k @ k.t())).abs()
    terms = strict * (k.abs() @ k.abs().t())
    seen = torch.exp(total)[:, None] * (k.abs() @ initial.abs().t())
    right = b[:, None] * (v.abs() + seen)
    size = inverse @ right
    carried = b[:, None] * torch.exp(total)[:, None] * (k.abs() @ off.t())
    return total, decay, size, inverse @ (EPS * (right + terms @ size) + carried)


def outputs(queries, keys, values, log_decay, beta, parents, initial, scale, normalize):
    """[T,H,128], of draft_reference.tree's `out`."""
    heads = values.shape[1]
    q, k = expanded(queries, keys, heads // keys.shape[1], scale, normalize)
    v, g, b, s = values.double(), log_decay.double(), beta.double(), initial.double()
    bound = torch.zeros(values.shape, dtype=torch.float64)
    for h in range(heads):
        total, decay, size, off = _writes(q[:, h], k[:, h], v[:, h], g[:, h], b[:, h], parents,
                                          s[h], torch.zeros_like(s[h]))
        look = decay * (q[:, h].abs() @ k[:, h].abs().t())
        read = torch.exp(total)[:, None] * (q[:, h].abs() @ s[h].abs().t())
        bound[:, h] = EPS * (read + look @ size) + look @ off
    return bound


def state(queries, keys, values, log_decay, beta, parents, initial, scale, normalize, node):
    """[H,128 value,128 key], of the state after `node`: 32 nodes of its path at a time."""
    heads = values.shape[1]
    _, k = expanded(queries, keys, heads // keys.shape[1], scale, normalize)
    v, g, b = values.double(), log_decay.double(), beta.double()
    path = ref.path(parents, node)
    bound = torch.zeros(initial.shape, dtype=torch.float64)
    now = initial.double().clone()
    for first in range(0, len(path), 32):
        at = path[first:first + 32]
        chain = list(range(-1, len(at) - 1))
        _, states = ref.tree(queries[at], keys[at], values[at], log_decay[at], beta[at], chain,
                             now, scale, normalize)
        for h in range(heads):
            total, decay, size, off = _writes(k[at, h], k[at, h], v[at, h], g[at, h], b[at, h],
                                              chain, now[h], bound[h])
            left = torch.exp(total[-1])
            weighted = (decay[-1][:, None] * k[at, h].abs())
            bound[h] = (left * (bound[h] + EPS * now[h].abs())
                        + (EPS * size + off).t() @ weighted)
        now = states[-1]
    return bound
