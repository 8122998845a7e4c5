"""Drafted trees and slot moves as a serving program runs them, against float64: prompts
into a pool, forks of their states, rounds of trees verified and paths committed, slots
freed and the live ones packed to the front, and single tokens after that.  Also the
example's answers by trees.

Tolerances as in tests/test_draft_tree_gpu.py: outputs 2^-9 + 2^-12 of their 2-norm from
the rounded float64 ones.  A state passes some 150 tokens in up to 8 calls; each call adds
2^-18 of it at most, and the earlier ones' errors decay with it: 2^-16."""

from __future__ import annotations

import importlib.util
import random
from pathlib import Path

import pytest
import torch

import delta_reference as delta
import draft_reference as ref
import gdn_state_codec as gdn

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -9 + 2.0 ** -12
HEADS, KEY_HEADS, LAYERS = 4, 2, 2


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def tokens(n, gen):
    """q, k, v, log decay, beta of n tokens on the CPU."""
    q, k = (torch.randn((n, KEY_HEADS, 128), generator=gen).bfloat16() for _ in range(2))
    v = torch.randn((n, HEADS, 128), generator=gen).bfloat16()
    g = -0.2 * torch.rand((n, HEADS), generator=gen)
    b = torch.sigmoid(torch.randn((n, HEADS), generator=gen)).bfloat16()
    return [q, k, v, g, b]


def close(got, want, bound, name):
    rounded = want.to(got.dtype) if got.dtype == torch.bfloat16 else want
    got, want = got.double().cpu(), rounded.double()
    off, size = float((got - want).norm()), float(want.norm())
    print(f"{name}: {off / size:.3g} (bound {bound:.3g})", flush=True)
    assert torch.isfinite(got).all() and off <= bound * size, name


@pytest.mark.parametrize("captured", [False, True])
def test_speculative_serving(device, captured):
    rng, gen = random.Random(5), torch.Generator().manual_seed(5)
    slots_of_pool = 12
    pool = [torch.randn((slots_of_pool, HEADS, 128, 128), generator=gen).to(device)
            for _ in range(LAYERS)]
    states = [dict() for _ in range(LAYERS)]  # slot -> float64 state

    lengths, slots = [70, 1, 33], [7, 2, 9]
    for layer in range(LAYERS):
        x = tokens(sum(lengths), gen)
        table = gdn.request_tables(ints(lengths, device), ints(slots, device), sum(lengths))
        gdn.gated_delta_prefill(*(t.to(device) for t in x), table, ints(slots, device),
                                pool[layer], resume=ints([0] * 3, device))
        _, final = delta.rule(*x, lengths, torch.zeros((3, HEADS, 128, 128)))
        states[layer].update(zip(slots, final))

    # Two samples more of the first prompt; the third slot is somebody's that is freed.
    gdn.copy_slots(pool, gdn.slot_moves(ints([7, 7, -1], device), ints([11, 4, 0], device),
                                        slots_of_pool))
    slots += [11, 4]
    for layer in range(LAYERS):
        states[layer][11] = states[layer][4] = states[layer][7]
        assert (pool[layer][0] == 0).all()

    # Rounds of trees of one total size, so that a captured round serves all of them.
    total = 40
    dev = [[t.to(device) for t in tokens(total, gen)] for _ in range(LAYERS)]
    parents, accepted = ints([0] * total, device), ints([0] * 5, device)
    sizes, ids = ints([0] * 5, device), ints(slots, device)
    outs = [torch.zeros((total, HEADS, 128), dtype=torch.bfloat16, device=device)
            for _ in range(LAYERS)]

    def work():
        table = gdn.request_tables(sizes, ids, total)
        for x, states, out in zip(dev, pool, outs):
            gdn.gated_delta_tree(*x, parents, table, ids, states, out=out)
            gdn.gated_delta_commit(*x[1:], parents, accepted, table, ids, states)

    graph = None
    for round_ in range(4):
        nodes = [rng.randint(0, 12) for _ in slots[:-1]]
        nodes = [min(n, 9) for n in nodes]
        nodes.append(rng.randint(0, total - sum(nodes)))
        trees = [ref.parents_of(rng.choice(["any", "chain", "branches"]), n, round_)
                 for n in nodes]
        takes = [rng.randint(-1, n - 1) for n in nodes]
        host = [tokens(total, gen) for _ in range(LAYERS)]
        for x, new in zip(dev, host):
            for t, value in zip(x, new):
                t.copy_(value)
        flat = [p for tree in trees for p in tree]
        parents.copy_(ints(flat + [0] * (total - len(flat)), device))
        accepted.copy_(ints(takes, device))
        sizes.copy_(ints(nodes, device))
        torch.cuda.synchronize()
        if captured and graph is None:
            saved = [t.clone() for t in pool]
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                work()  # warms up, on a pool that is put back
            stream.synchronize()
            for t, old in zip(pool, saved):
                t.copy_(old)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                work()
        graph.replay() if captured else work()
        torch.cuda.synchronize()
        for layer in range(LAYERS):
            at = 0
            for slot, tree, take in zip(slots, trees, takes):
                part = [t[at:at + len(tree)] for t in host[layer]]
                want, after = ref.tree(*part, tree, states[layer][slot])
                if tree:
                    close(outs[layer][at:at + len(tree)], want, BF16, f"round {round_}")
                if take >= 0:
                    states[layer][slot] = after[take]
                at += len(tree)

    # One sample ends; the others are packed to the front, and go on with single tokens.
    slots.remove(11)
    live = [int(i in slots) for i in range(slots_of_pool)]
    packed = gdn.compaction_moves(ints(live, device))
    gdn.copy_slots(pool, packed.moves)
    place = packed.placed.tolist()
    assert packed.count.tolist() == [4] and sorted(place[s] for s in slots) == [0, 1, 2, 3]
    ids = packed.placed[ints(slots, device).long()].contiguous()
    for layer in range(LAYERS):
        x = tokens(4, gen)
        out = gdn.gated_delta_step(*(t.to(device) for t in x), pool[layer], ids)
        want, final = delta.rule(*x, [1] * 4, torch.stack([states[layer][s] for s in slots]))
        close(out, want, BF16, "single tokens")
        close(pool[layer][ids.long()], final, 2.0 ** -16, "states")


def test_the_examples_answers_by_trees(device):
    path = Path(__file__).resolve().parents[1] / "examples" / "gated_delta_net.py"
    spec = importlib.util.spec_from_file_location("gated_delta_net", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(3)
    net = example.Net().to(device)
    off = example.serve(net, [40, 1, 130], 10, device, torch.Generator().manual_seed(3))
    print(off, flush=True)
    # As the answers decoded token by token (tests/test_layer_example_gpu.py).
    assert off["decoded by trees"] <= 2.0 ** -5 and off["decoded"] <= 2.0 ** -5
