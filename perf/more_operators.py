"""Drafted tokens and slot moves on the state pool: what is measured, with plain forms.

Speculative decoding of a gated-delta-net layer: the rule over a tree of drafted
tokens of each request, read from its cached state without changing it; and the
state advanced along the accepted path.  And what a serving program does to the
slots of such a cache: copying, forking and reordering them, clearing freed ones,
and packing the live ones to the front.

``run`` computes the plain forms with elementary torch operations in fp32 where
``own`` is false, and calls the package's operators where it is true.  ``exact``
evaluates the definitions in float64, node by node and slot by slot.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DIM = 128
CHUNK = 64
MOST_NODES = 64
L2_EPS = 1e-6
SCALE = DIM ** -0.5

# Bytes of one head's encoded slot: int8 codes, fp32 smoothing and scales, fp16
# compensators, the window's fp32 decays, fp16 keys and corrections, int32 positions.
ENCODED = (("i8", DIM * DIM), ("f32", DIM), ("f32", DIM), ("f16", DIM * 4), ("f16", DIM * 4),
           ("f32", 16), ("f16", 16 * DIM), ("f16", 16 * DIM), ("i32", 8))
CELL = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1, "i32": 4}


def listed() -> list[dict]:
    return [
        # A chain of 5 drafted tokens of a single request: 32 heads, fp32 states.
        {"name": "tree_1", "kind": "tree", "requests": 1, "longest": 5, "shape": "chain",
         "heads": 32, "key_heads": 16, "pool": "f32", "padded": 0, "even": True},
        # A decode batch of 64 requests with a bushy tree of 16 nodes each, some padding.
        {"name": "tree_64", "kind": "tree", "requests": 64, "longest": 16, "shape": "bushy",
         "heads": 32, "key_heads": 16, "pool": "f32", "padded": 3, "even": True},
        # 256 requests with trees of 0 to 48 nodes on a bf16 pool.
        {"name": "tree_ragged", "kind": "tree", "requests": 256, "longest": 48,
         "shape": "bushy", "heads": 32, "key_heads": 16, "pool": "bf16", "padded": 5,
         "even": False},
        # The longest drafts: 128 requests with a chain of 64 tokens each.
        {"name": "tree_chains", "kind": "tree", "requests": 128, "longest": 64,
         "shape": "chain", "heads": 32, "key_heads": 16, "pool": "f32", "padded": 0,
         "even": True},
        # The accepted tokens of that single request.
        {"name": "commit_1", "kind": "commit", "requests": 1, "longest": 5, "shape": "chain",
         "heads": 32, "key_heads": 16, "pool": "f32", "padded": 0, "even": True},
        # The accepted paths of 256 requests with trees of 16 nodes; some accept nothing.
        {"name": "commit_256", "kind": "commit", "requests": 256, "longest": 16,
         "shape": "bushy", "heads": 32, "key_heads": 16, "pool": "f32", "padded": 5,
         "even": True},
        # Long accepted paths out of chains of 64, on a bf16 pool.
        {"name": "commit_chains", "kind": "commit", "requests": 128, "longest": 64,
         "shape": "chain", "heads": 32, "key_heads": 16, "pool": "bf16", "padded": 0,
         "even": True},
        # One prompt's state forked to 4 samples of it, one layer.
        {"name": "fork_1", "kind": "move", "how": "fork", "pairs": 4, "slots": 16, "layers": 1,
         "heads": 32, "cells": "f32", "cleared": 0},
        # A beam search step: 96 slots take each other's states in 8 layers.
        {"name": "beams_96", "kind": "move", "how": "beams", "pairs": 96, "slots": 100,
         "layers": 8, "heads": 32, "cells": "f32", "cleared": 0},
        # Encoded slots (codes, scales, compensators and their window): prefixes forked,
        # and freed slots cleared.
        {"name": "fork_encoded", "kind": "move", "how": "fork", "pairs": 300, "slots": 700,
         "layers": 1, "heads": 32, "cells": "encoded", "cleared": 50},
        # A pool of 256 slots with 60% of them live, packed to the front in 4 layers.
        {"name": "compact_256", "kind": "compact", "slots": 256, "live": 154, "layers": 4,
         "heads": 32, "cells": "bf16"},
    ]


def draw(rng) -> dict:
    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(["tree", "tree", "commit", "commit", "move", "compact"])
    if kind in ("tree", "commit"):
        longest = size(1, MOST_NODES)
        requests = size(1, min(256, 8192 // longest))
        key_heads = rng.choice([1, 2, 4, 8, 16])
        heads = key_heads * rng.choice([1, 2, 2, 4] if key_heads < 16 else [1, 2])
        return {"kind": kind, "requests": requests, "longest": longest,
                "shape": rng.choice(["chain", "bushy", "bushy", "wide"]), "heads": heads,
                "key_heads": key_heads, "pool": rng.choice(["f32", "bf16"]),
                "padded": rng.randint(0, requests // 8), "even": rng.random() < 0.5,
                "draw": rng.randrange(1 << 20)}
    layers, heads = size(1, 12), size(1, 32)
    if kind == "move":
        cells = rng.choice(["f32", "bf16", "encoded"])
        most = max(1, min(1024, (1250 << 20) // (layers * _slot_bytes(cells, heads))))
        pairs = size(1, most)
        how = rng.choice(["fork", "beams", "permute"])
        return {"kind": kind, "how": how, "pairs": pairs,
                "slots": pairs * (2 if how == "fork" else 1) + rng.randint(1, 5),
                "layers": layers, "heads": heads, "cells": cells,
                "cleared": rng.randint(0, pairs // 4), "draw": rng.randrange(1 << 20)}
    cells = rng.choice(["f32", "bf16", "encoded"])
    slots = size(2, max(2, min(2048, (2500 << 20) // (layers * _slot_bytes(cells, heads)))))
    return {"kind": kind, "slots": slots, "live": rng.randint(0, slots), "layers": layers,
            "heads": heads, "cells": cells, "draw": rng.randrange(1 << 20)}


# ------------------------------------------------------------- a case's shapes

def _slot_bytes(cells: str, heads: int) -> int:
    if cells == "encoded":
        return heads * sum(n * CELL[t] for t, n in ENCODED)
    return heads * DIM * DIM * CELL[cells]


def _parents(rng, nodes: int, shape: str) -> list[int]:
    """Each node's parent, an earlier node or -1: a chain; a bushy tree below the last
    sampled token, as the likeliest continuations give; or many short branches, some of
    them from the cached state."""
    if shape == "chain":
        return list(range(-1, nodes - 1))
    if shape == "wide":
        return [-1 if i == 0 or rng.random() < 0.3 else rng.randint(max(0, i // 3 - 1), i // 2)
                if i > 1 else 0 for i in range(nodes)]
    return [-1 if i == 0 else rng.randint(max(0, i - 6), i - 1) for i in range(nodes)]


def _trees(case: dict) -> list[tuple]:
    """(parents, accepted node or -1, padding) of each request.  Ragged batches have an
    empty and a one-node tree."""
    rng = random.Random(case.get("draw", 3) * 8191 + case["requests"])
    n, longest = case["requests"], case["longest"]
    counts = [longest] * n
    if not case["even"]:
        counts = [longest] + [rng.randint(0, longest) for _ in range(n - 1)]
        if n > 3:
            counts[1], counts[2] = 0, 1
    trees = []
    for i, nodes in enumerate(counts):
        accepted = rng.randint(nodes // 2 - 1 if case["shape"] == "chain" else -1, nodes - 1)
        trees.append((_parents(rng, nodes, case["shape"]), accepted, i >= n - case["padded"]))
    rng.shuffle(trees)
    return trees


def _path(parents: list[int], node: int) -> list[int]:
    path = []
    while node >= 0:
        path.append(node)
        node = parents[node]
    return path[::-1]


# ------------------------------------------------------------------- inputs

def _device() -> torch.device:
    return torch.device("cuda", torch.cuda.current_device())


def _dtype(name: str) -> torch.dtype:
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
            "i8": torch.int8, "i32": torch.int32}[name]


def _tokens_of_a_layer(tokens, heads, key_heads, gen, dev):
    """Queries, keys and values as slices of one fused projection, the log decays and
    the write strengths of one layer."""
    mixed = torch.randn((tokens, (2 * key_heads + heads) * DIM), generator=gen,
                        device=dev).to(torch.bfloat16)
    q = mixed[:, :key_heads * DIM].view(tokens, key_heads, DIM)
    k = mixed[:, key_heads * DIM:2 * key_heads * DIM].view(tokens, key_heads, DIM)
    v = mixed[:, 2 * key_heads * DIM:].view(tokens, heads, DIM)
    rate = torch.exp(torch.rand((1, heads), generator=gen, device=dev) * 6.0 - 6.0)
    noise = torch.randn((tokens, heads), generator=gen, device=dev)
    log_decay = -rate * torch.nn.functional.softplus(noise)
    beta = torch.sigmoid(torch.randn((tokens, heads), generator=gen, device=dev))
    return q, k, v, log_decay, beta.to(torch.bfloat16)


def _tables(lengths: list[int], slots: list[int], dev):
    """offsets [N+1], chunk_offsets [N+1], chunks [rows,4], order [N] (int32)."""
    offsets, first, chunks = [0], [0], []
    for r, length in enumerate(lengths):
        begin = offsets[-1]
        chunks += [[r, t, min(CHUNK, begin + length - t), slots[r]]
                   for t in range(begin, begin + length, CHUNK)]
        offsets.append(begin + length)
        first.append(len(chunks))
    order = sorted(range(len(lengths)), key=lambda r: first[r] - first[r + 1])
    chunks += [[-1, 0, 0, -1]] * (offsets[-1] // CHUNK + len(lengths) - len(chunks))
    return tuple(torch.tensor(x, dtype=torch.int32, device=dev)
                 for x in (offsets, first, chunks, order))


def _prepare_trees(case: dict, seed: int, gen, dev) -> dict:
    rng = random.Random(seed)
    trees = _trees(case)
    rng.shuffle(trees)
    n, h, hk = len(trees), case["heads"], case["key_heads"]
    lens = [len(t[0]) for t in trees]
    total = sum(lens)
    q, k, v, log_decay, beta = _tokens_of_a_layer(total, h, hk, gen, dev)
    room = rng.sample(range(n + 3), n)
    slots = [-1 if t[2] else slot for t, slot in zip(trees, room)]

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    pool = torch.empty((n + 3, h, DIM, DIM), dtype=_dtype(case["pool"]), device=dev)
    for slot in pool:  # one at a time: no fp32 copy of the whole
        slot.copy_(0.1 * torch.randn(slot.shape, generator=gen, device=dev))
    return {"kind": case["kind"], "lens": lens, "q": q, "k": k, "v": v,
            "log_decay": log_decay, "beta": beta,
            "parents": ints([p for t in trees for p in t[0]]),
            "accepted": ints([t[1] for t in trees]), "slots": ints(slots),
            "tables": _tables(lens, slots, dev), "pool": pool,
            "out": torch.zeros((total, h, DIM), dtype=torch.bfloat16, device=dev)}


def _buffers(case: dict, gen, dev) -> list:
    """A cache's tensors, one row a slot: a dense pool of each layer, or the nine
    buffers of encoded slots."""
    slots, heads = case["slots"], case["heads"]
    if case["cells"] != "encoded":
        dtype = _dtype(case["cells"])
        made = [torch.empty((slots, heads, DIM, DIM), dtype=dtype, device=dev)
                for _ in range(case["layers"])]
    else:
        made = [torch.empty((slots, heads, n), dtype=_dtype(t), device=dev)
                for _ in range(case["layers"]) for t, n in ENCODED]
    for t in made:
        if t.dtype in (torch.int8, torch.int32):
            t.random_(-127, 128, generator=gen)
        else:
            t.normal_(generator=gen)
    return made


def prepare(case: dict, seed: int) -> dict:
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind = case["kind"]
    if kind in ("tree", "commit"):
        return _prepare_trees(case, seed, gen, dev)
    rng = random.Random(seed)
    slots = case["slots"]
    state = {"kind": kind, "buffers": _buffers(case, gen, dev), "slots": slots}
    if kind == "compact":
        live = set(rng.sample(range(slots), case["live"]))
        state["live"] = torch.tensor([int(i in live) for i in range(slots)],
                                     dtype=torch.int32, device=dev)
        return state
    pairs = case["pairs"]
    if case["how"] == "fork":  # a few prefixes, each to several slots that are free
        place = rng.sample(range(slots), slots)
        targets, kept = place[:pairs], place[pairs:]
        few = kept[:max(1, pairs // 4)]
        sources = [rng.choice(few) for _ in targets]
    else:
        targets = rng.sample(range(slots), pairs)
        sources = [rng.choice(targets) for _ in targets]
        if case["how"] == "permute":
            sources = rng.sample(targets, pairs)
    for i in rng.sample(range(pairs), case["cleared"]):
        sources[i] = -1
    state["sources"], state["targets"] = (
        torch.tensor(x, dtype=torch.int32, device=dev) for x in (sources, targets))
    return state


# ----------------------------------------------------------- the plain forms

def _unit(x: torch.Tensor) -> torch.Tensor:
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + L2_EPS)


def _side_by_side(s: dict):
    """Requests side by side: their token rows [N,W] (-1 past each tree's end), and
    whether node j is node i or above it, [N,W,W]."""
    dev = s["q"].device
    length = torch.tensor(s["lens"], device=dev)
    width = max(1, max(s["lens"]))
    at = torch.arange(width, device=dev)[None, :]
    start = torch.cumsum(length, 0) - length
    index = torch.where(at < length[:, None], start[:, None] + at, -1)
    live = index >= 0
    parent = torch.where(live, s["parents"].long()[index.clamp(min=0)], -1)
    step = (parent[:, :, None] == at[:, None, :]).float()
    above = torch.eye(width, device=dev) + step
    for _ in range(max(0, (width - 1).bit_length() - 1)):  # paths of up to 2, 4, 8 .. steps
        step = torch.matmul(step, step)
        above = above + torch.matmul(above, step)
    return index, live, above > 0.5


def _plain_tree_writes(s: dict):
    """Each node's write u and what its reads need: [N,H,W,...] in fp32."""
    index, live, above = _side_by_side(s)
    n, width = index.shape
    h = s["v"].shape[1]
    group = h // s["q"].shape[1]
    at = index.clamp(min=0)

    def rows(x):  # [T,H,D] -> [N,H,W,D], zeros past each tree's end
        x = torch.where(live[..., None, None], x[at], torch.zeros((), device=x.device))
        return x.permute(0, 2, 1, 3).contiguous()

    q = rows((_unit(s["q"].float()) * SCALE).repeat_interleave(group, 1))
    k = rows(_unit(s["k"].float()).repeat_interleave(group, 1))
    v, b, g = rows(s["v"].float()), rows(s["beta"].float()[..., None]), \
        rows(s["log_decay"][..., None])
    mask = above[:, None]
    total = torch.matmul(mask.float(), g)  # log decays from the state to the node
    decay = torch.exp((total - total.transpose(-1, -2)).masked_fill(~mask, -math.inf))
    slots = s["slots"].long().clamp(min=0)
    state = s["pool"][slots].float().transpose(-1, -2).contiguous()  # [N,H,key,value]
    kt = k.transpose(-1, -2).contiguous()
    step = -b * decay * torch.matmul(k, kt) * (1.0 - torch.eye(width, device=k.device))
    u = b * (v - torch.exp(total) * torch.matmul(k, state))
    for _ in range(max(1, (width - 1).bit_length())):  # (1 + A)(1 + A^2)(1 + A^4) ..
        u = u + torch.matmul(step, u)
        step = torch.matmul(step, step)
    return index, live, mask, q, k, kt, total, decay, state, u


def _plain_tree(s: dict):
    index, live, _, q, _, kt, total, decay, state, u = _plain_tree_writes(s)
    out = torch.exp(total) * torch.matmul(q, state) + torch.matmul(decay * torch.matmul(q, kt), u)
    kept = live & (s["slots"] >= 0)[:, None]
    s["out"][index[kept]] = out.permute(0, 2, 1, 3)[kept].to(s["out"].dtype)
    return {"out": s["out"]}


def _plain_commit(s: dict):
    _, _, mask, _, k, _, total, decay, state, u = _plain_tree_writes(s)
    node = s["accepted"].long()
    moved = torch.nonzero((node >= 0) & (s["slots"] >= 0)).reshape(-1)
    node, slots = node[moved], s["slots"].long()[moved]
    at = (moved, slice(None), node)
    weight = decay[at] * mask[moved, 0, node][:, None].float()  # [M,H,W]
    after = (torch.exp(total[at])[..., None] * state[moved]
             + torch.matmul((k[moved] * weight[..., None]).transpose(-1, -2).contiguous(),
                            u[moved]))
    s["pool"][slots] = after.transpose(-1, -2).to(s["pool"].dtype)
    return {"pool": s["pool"]}


def _plain_move(buffers, sources, targets):
    """All pairs at once: every source as it was; a source of -1 gives zeros."""
    sources, targets = sources.long(), targets.long()
    for t in buffers:
        rows = t[sources.clamp(min=0)]
        empty = (sources < 0).reshape(-1, *[1] * (t.dim() - 1))
        t[targets] = rows.masked_fill(empty, 0)


def _plain_compact(s: dict):
    """Live slots behind the first `count` move into free ones among them, in order."""
    live = s["live"] != 0
    at = torch.arange(live.numel(), device=live.device)
    count = live.sum()
    targets = torch.nonzero(~live & (at < count)).reshape(-1)
    sources = torch.nonzero(live & (at >= count)).reshape(-1)
    placed = torch.where(live, at, -1)
    placed[sources] = targets
    _plain_move(s["buffers"], sources, targets)
    return {"placed": placed.to(torch.int32), "count": count.to(torch.int32).reshape(1),
            "buffers": s["buffers"]}


# ------------------------------------------------------------ the operators

def _package():
    path = str(Path(__file__).resolve().parents[1] / "gdn-state-codec_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gdn_state_codec

    return gdn_state_codec


def _own(s: dict):
    package = _package()
    kind = s["kind"]
    if kind == "tree":
        package.gated_delta_tree(s["q"], s["k"], s["v"], s["log_decay"], s["beta"],
                                 s["parents"], package.RequestTables(*s["tables"]), s["slots"],
                                 s["pool"], out=s["out"])
        return {"out": s["out"]}
    if kind == "commit":
        package.gated_delta_commit(s["k"], s["v"], s["log_decay"], s["beta"], s["parents"],
                                   s["accepted"], package.RequestTables(*s["tables"]),
                                   s["slots"], s["pool"])
        return {"pool": s["pool"]}
    if kind == "move":
        moves = package.slot_moves(s["sources"], s["targets"], s["slots"])
        package.copy_slots(s["buffers"], moves)
        return {"buffers": s["buffers"]}
    packed = package.compaction_moves(s["live"])
    package.copy_slots(s["buffers"], packed.moves)
    return {"placed": packed.placed, "count": packed.count, "buffers": s["buffers"]}


def run(state: dict):
    if own:
        return _own(state)
    kind = state["kind"]
    if kind == "tree":
        return _plain_tree(state)
    if kind == "commit":
        return _plain_commit(state)
    if kind == "move":
        _plain_move(state["buffers"], state["sources"], state["targets"])
        return {"buffers": state["buffers"]}
    return _plain_compact(state)


# -------------------------------------------------------------- 64-bit values

def _unit64(x: torch.Tensor) -> torch.Tensor:
    return x * ((x * x).sum(-1, keepdim=True) + L2_EPS) ** -0.5


def _exact_trees(s: dict):
    """Node by node, from the state its parent leaves: S' = a S; S = S' + b (v - S' k) k^T;
    o = S q.  A few requests at a time, whose nodes' states are all kept."""
    h = s["v"].shape[1]
    group = h // s["q"].shape[1]
    starts = [0]
    for length in s["lens"]:
        starts.append(starts[-1] + length)
    parents, slots = s["parents"].tolist(), s["slots"].tolist()
    accepted = s["accepted"].tolist()
    out, pool = s["out"].double(), s["pool"].double() if s["kind"] == "commit" else None
    each = max(1, (6 << 30) // (max(1, max(s["lens"])) * h * DIM * DIM * 8))
    live = [r for r, slot in enumerate(slots) if slot >= 0 and s["lens"][r]]
    dev = s["q"].device
    for first in range(0, len(live), each):
        some = live[first:first + each]
        width = max(s["lens"][r] for r in some)
        begin = torch.stack([s["pool"][slots[r]] for r in some]).double()
        states = torch.empty((width + 1, *begin.shape), dtype=torch.float64, device=dev)
        states[0] = begin
        for i in range(width):
            rows = [j for j, r in enumerate(some) if i < s["lens"][r]]
            at = torch.tensor([starts[some[j]] + i for j in rows], device=dev)
            above = torch.tensor([parents[starts[some[j]] + i] + 1 for j in rows], device=dev)
            rows = torch.tensor(rows, device=dev)
            k = _unit64(s["k"][at].double()).repeat_interleave(group, 1)
            q = (_unit64(s["q"][at].double()) * SCALE).repeat_interleave(group, 1)
            state = states[above, rows] * torch.exp(s["log_decay"][at].double())[..., None, None]
            error = s["v"][at].double() - torch.matmul(state, k[..., None])[..., 0]
            write = s["beta"][at].double()[..., None] * error
            state = state + write[..., :, None] * k[..., None, :]
            states[i + 1, rows] = state
            out[at] = torch.matmul(state, q[..., None])[..., 0]
        if pool is not None:
            for j, r in enumerate(some):
                if accepted[r] >= 0:
                    pool[slots[r]] = states[accepted[r] + 1, j]
    return {"out": out} if pool is None else {"pool": pool}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if s["kind"] in ("tree", "commit"):
        return _exact_trees(s)
    if s["kind"] == "compact":
        live = s["live"].tolist()
        count = sum(1 for x in live if x)
        free = [i for i in range(count) if not live[i]]
        late = [i for i in range(count, len(live)) if live[i]]
        to = dict(zip(late, free))
        placed = [to.get(i, i) if x else -1 for i, x in enumerate(live)]
        pairs = list(to.items())
    else:
        pairs = list(zip(s["sources"].tolist(), s["targets"].tolist()))
    after = []
    for t in s["buffers"]:
        new = t.clone()
        for source, target in pairs:
            if source < 0:
                new[target] = 0
            else:
                new[target] = t[source]
        after.append(new)
    if s["kind"] == "move":
        return {"buffers": after}
    return {"placed": torch.tensor(placed, dtype=torch.int32),
            "count": torch.tensor([count], dtype=torch.int32), "buffers": after}


# ------------------------------------------------------------------ the floor

def work(case: dict) -> dict:
    kind = case["kind"]
    if kind in ("tree", "commit"):
        h, hk = case["heads"], case["key_heads"]
        state = h * DIM * DIM * CELL[case["pool"]]
        trees = [t for t in _trees(case) if not t[2]]
        # keys, values, log decays, write strengths and the parents of a node
        node = 2 * hk * DIM + 2 * h * DIM + 6 * h + 4
        if kind == "tree":  # each state once, the queries too, and the outputs
            nodes = sum(len(t[0]) for t in trees)
            each = node + 2 * hk * DIM + 2 * h * DIM
            return {"bytes": sum(1 for t in trees if t[0]) * state + nodes * each,
                    "flops": 4 * nodes * h * DIM * DIM}
        # the states of requests that accept something, read and written
        nodes = sum(len(_path(t[0], t[1])) for t in trees)
        return {"bytes": 2 * sum(1 for t in trees if t[1] >= 0) * state + nodes * node,
                "flops": 4 * nodes * h * DIM * DIM}
    slot = _slot_bytes(case["cells"], case["heads"]) * case["layers"]
    if kind == "move":  # each different source read once, each target written once
        rng, pairs, cleared = random.Random(1), case["pairs"], case["cleared"]
        left = pairs - cleared
        if case["how"] == "permute":
            read = left
        else:
            few = max(1, pairs // 4) if case["how"] == "fork" else pairs
            read = min(left, len({rng.randrange(few) for _ in range(left)}))
        return {"bytes": slot * (read + pairs) + 8 * pairs, "flops": 0}
    # about live x free / slots of the live ones lie behind the first `live`
    moved = case["live"] * (case["slots"] - case["live"]) // case["slots"]
    return {"bytes": 2 * slot * moved + 8 * case["slots"] + 4, "flops": 0}
