"""Moves between the slots of a state cache (slot_moves, compaction_moves, copy_slots,
GdnStateCodecRuntime.fork) on the GPU against their definitions, bit for bit."""

from __future__ import annotations

import random

import pytest
import torch

import draft_reference as ref
import gdn_state_codec as gdn
from gdn_state_codec import window

pytestmark = pytest.mark.gpu


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def bits(t):
    """Rows as bytes, so that NaNs compare too."""
    return t.contiguous().view(t.shape[0], -1).view(torch.uint8).cpu()


def filled(shape, dtype, device, seed=5):
    gen = torch.Generator().manual_seed(seed)
    if dtype.is_floating_point:
        return torch.randn(shape, generator=gen).to(dtype).to(device)
    return torch.randint(-128, 128, shape, generator=gen).to(dtype).to(device)


def check(device, sources, targets, slots, buffers):
    want = [ref.moved(bits(t), sources, targets) for t in buffers]
    gdn.copy_slots(buffers, gdn.slot_moves(ints(sources, device), ints(targets, device), slots))
    for got, expected in zip(buffers, want):
        assert torch.equal(bits(got), expected)


def _pairs(kind, slots, n, rng):
    if kind == "fork":
        order = rng.sample(range(slots), slots)
        return [rng.choice(order[n:] or order) for _ in range(n)], order[:n]
    if kind == "beams":
        targets = rng.sample(range(slots), n)
        return [rng.choice(targets) for _ in targets], targets
    if kind == "permute":
        targets = rng.sample(range(slots), n)
        return rng.sample(targets, n), targets
    if kind == "rotate":  # one cycle through all of them
        targets = rng.sample(range(slots), n)
        return targets[1:] + targets[:1], targets
    if kind == "shift":  # one chain
        targets = rng.sample(range(slots), n)
        return targets[1:] + [(set(range(slots)) - set(targets)).pop()], targets
    if kind == "same":
        targets = rng.sample(range(slots), n)
        return list(targets), targets
    # anything: padding, sources and targets outside, cleared and repeated targets
    return ([rng.randint(-3, slots + 1) for _ in range(n)],
            [rng.randint(-3, slots + 1) for _ in range(n)])


KINDS = ("fork", "beams", "permute", "rotate", "shift", "same", "any")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pairs,slots", [(1, 2), (2, 3), (3, 9), (7, 8), (8, 9), (9, 30),
                                         (64, 65), (100, 333), (257, 300), (1000, 1001)])
def test_moves(device, kind, pairs, slots):
    for seed in range(3):
        rng = random.Random(100 * pairs + seed)
        sources, targets = _pairs(kind, slots, pairs, rng)
        check(device, sources, targets, slots, [filled((slots, 24), torch.float32, device, seed)])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pairs", [1023, 1024, 1025, 4095, 4096])
def test_many_pairs(device, kind, pairs):
    sources, targets = _pairs(kind, 5000, pairs, random.Random(pairs))
    check(device, sources, targets, 5000, [filled((5000, 12), torch.int32, device)])


def test_cycles_of_every_length_and_trees_into_them(device):
    rng = random.Random(3)
    slots = list(range(700))
    rng.shuffle(slots)
    sources, targets = [], []
    for length in range(1, 25):
        cycle = [slots.pop() for _ in range(length)]
        sources += cycle[1:] + cycle[:1]
        targets += cycle
        for _ in range(3):  # chains that read the cycle's slots
            at = rng.choice(cycle)
            for _ in range(rng.randint(1, 5)):
                new = slots.pop()
                sources.append(at)
                targets.append(new)
                at = new
    order = rng.sample(range(len(sources)), len(sources))
    check(device, [sources[i] for i in order], [targets[i] for i in order], 700,
          [filled((700, 40), torch.float32, device)])


def test_swap(device):
    check(device, [3, 1], [1, 3], 5, [filled((5, 2, 128, 128), torch.bfloat16, device)])


@pytest.mark.parametrize("shape,dtype", [
    ((1,), torch.int8), ((3,), torch.int8), ((17,), torch.int8), ((4096,), torch.int8),
    ((4097,), torch.int8), ((1,), torch.int32), ((5,), torch.float32), ((8,), torch.int32),
    ((3, 7), torch.bfloat16), ((2, 128, 4), torch.float16), ((1, 128, 128), torch.float32),
    ((3, 128, 128), torch.bfloat16), ((5000,), torch.float64), ((0,), torch.float32), ((), torch.int32)])
def test_rows_of_any_size(device, shape, dtype):
    sources, targets = _pairs("beams", 23, 20, random.Random(11))
    sources[4] = sources[9] = -1
    buffer = filled((23, *shape), dtype, device)
    if buffer.numel():
        check(device, sources, targets, 23, [buffer])
    else:
        gdn.copy_slots(buffer, gdn.slot_moves(ints(sources, device), ints(targets, device), 23))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size,dtype,more", [(270001, torch.int8, 0), (275001, torch.float32, 0),
                                             (1050004, torch.float32, 0),
                                             (5000, torch.float32, 70)])
def test_many_workgroups(device, kind, size, dtype, more):
    """Rows of 1,024 and more workgroups, in units of 1, 4 and 16 bytes, alone and in many
    buffers; cleared slots beside the moved ones, more rows than are carried out together."""
    sources, targets = _pairs(kind, 30, 25, random.Random(size))
    sources[3] = sources[20] = -1
    check(device, sources, targets, 30,
          [filled((30, size), dtype, device, i) for i in range(1 + more)])


def test_rows_that_start_at_any_byte(device):
    """A buffer that is a slice: 4-byte and 1-byte aligned, the bytes around it untouched."""
    for dtype, skip in ((torch.float32, 1), (torch.int8, 3), (torch.int8, 4)):
        whole = filled((skip + 9 * 32 + 5,), dtype, device)
        before = whole.clone()
        part = whole[skip:skip + 9 * 32].view(9, 32)
        check(device, [1, 2, 0, -1], [0, 1, 2, 8], 9, [part])
        assert torch.equal(whole[:skip], before[:skip])
        assert torch.equal(whole[skip + 288:], before[skip + 288:])


@pytest.mark.parametrize("count", [1, 2, 9, 63, 64, 65, 130])
def test_many_buffers(device, count):
    sources, targets = _pairs("beams", 12, 10, random.Random(count))
    sizes = [(1,), (16,), (33,), (4, 100), (1030,)]
    types = [torch.float32, torch.int8, torch.bfloat16]
    check(device, sources, targets, 12,
          [filled((12, *sizes[i % 5]), types[i % 3], device, i) for i in range(count)])


def test_nan_and_infinity_are_copied_as_they_are(device):
    buffer = filled((6, 64), torch.float32, device)
    buffer[2, 5], buffer[2, 6], buffer[2, 7] = float("nan"), float("inf"), -0.0
    check(device, [2, 0], [4, 2], 6, [buffer])


def test_into_other_buffers(device):
    """From one cache into another; the first stays as it is, cycles and all."""
    for kind in KINDS:
        sources, targets = _pairs(kind, 40, 31, random.Random(7))
        held = [filled((40, 3, 50), torch.float32, device), filled((40, 7), torch.int8, device)]
        into = [filled(t.shape, t.dtype, device, 9) for t in held]
        before = [bits(t) for t in held]
        want = []
        for old, new in zip(before, map(bits, into)):
            after = new.clone()
            for s, t in zip(sources, targets):
                if 0 <= t < 40 and -1 <= s < 40:
                    after[t] = old[s] if s >= 0 else 0
            want.append(after)
        gdn.copy_slots(held, gdn.slot_moves(ints(sources, device), ints(targets, device), 40),
                       into=into)
        for got, expected in zip(into, want):
            assert torch.equal(bits(got), expected)
        for t, expected in zip(held, before):
            assert torch.equal(bits(t), expected)


def test_slots_past_four_gibibytes(device):
    pool = torch.empty((4600, 16, 128, 128), device=device)  # 4.8 GB
    rows = {i: filled((16, 128, 128), torch.float32, device, i) for i in (0, 4599, 4590)}
    for i, row in rows.items():
        pool[i] = row
    moves = gdn.slot_moves(ints([4599, 0, -1, 4590], device), ints([0, 4599, 4590, 7], device),
                           4600)
    gdn.copy_slots(pool, moves)
    assert torch.equal(pool[0], rows[4599]) and torch.equal(pool[4599], rows[0])
    assert torch.equal(pool[7], rows[4590]) and (pool[4590] == 0).all()


# --------------------------------------------------------------- compaction

def _live(kind, slots, rng):
    return {"none": [0] * slots, "all": [1] * slots,
            "front": [int(i < slots // 2) for i in range(slots)],
            "back": [int(i >= slots // 2) for i in range(slots)],
            "few": [int(rng.random() < 0.1) for _ in range(slots)],
            "any": [rng.choice([0, 0, 1, -1, 7]) for _ in range(slots)],
            "most": [int(rng.random() < 0.9) for _ in range(slots)]}[kind]


@pytest.mark.parametrize("kind", ["none", "all", "front", "back", "few", "any", "most"])
@pytest.mark.parametrize("slots", [1, 2, 3, 64, 257, 1023, 1024, 1025, 5000, 65536])
def test_compaction(device, kind, slots):
    live = _live(kind, slots, random.Random(slots))
    sources, targets, placed, count = ref.compacted(live)
    buffers = [filled((slots, 6), torch.int32, device), filled((slots, 5), torch.int8, device)]
    want = [ref.moved(bits(t), sources, targets) for t in buffers]
    packed = gdn.compaction_moves(ints(live, device))
    gdn.copy_slots(buffers, packed.moves)
    assert packed.placed.cpu().tolist() == placed and packed.count.cpu().tolist() == [count]
    assert packed.placed.dtype == packed.count.dtype == torch.int32
    for got, expected in zip(buffers, want):
        assert torch.equal(bits(got), expected)


# ------------------------------------------------------ together, and the runtime

def test_moves_serve_many_calls_and_replays(device):
    """One plan for several caches, on another stream; a captured plan and copy replay
    with other pairs each time."""
    sources, targets = _pairs("beams", 50, 40, random.Random(1))
    src, dst = ints(sources, device), ints(targets, device)
    layers = [filled((50, 2, 16, 16), torch.float32, device, i) for i in range(3)]
    want = [ref.moved(bits(t), sources, targets) for t in layers]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        moves = gdn.slot_moves(src, dst, 50)
        for t in layers:
            gdn.copy_slots(t, moves)
    stream.synchronize()
    assert all(torch.equal(bits(t), x) for t, x in zip(layers, want))
    live = ints([0] * 50, device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gdn.copy_slots(layers, gdn.slot_moves(src, dst, 50))
        packed = gdn.compaction_moves(live)
        gdn.copy_slots(layers, packed.moves)
    for take in range(3):
        rng = random.Random(take)
        sources, targets = _pairs("any" if take else "rotate", 50, 40, rng)
        alive = _live("any", 50, rng)
        src.copy_(ints(sources, device))
        dst.copy_(ints(targets, device))
        live.copy_(ints(alive, device))
        late, free, placed, _ = ref.compacted(alive)
        want = [ref.moved(ref.moved(bits(t), sources, targets), late, free) for t in layers]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bits(t), x) for t, x in zip(layers, want))
        assert packed.placed.cpu().tolist() == placed


def test_encoded_slots(device):
    """The nine buffers of a window slot of 6 x 4 states, in one call."""
    slot = window.WindowSlot.allocate(24, device)
    rows = slot.slot_rows(4)
    assert len(rows) == 9 and all(t.shape[:2] == (6, 4) for t in rows)
    for i, t in enumerate(rows):
        t.copy_(filled(t.shape, t.dtype, device, i))
    check(device, [0, 5, 0, -1], [5, 0, 2, 3], 6, rows)
    assert torch.equal(slot.positions.view(6, 4, 8), rows[8])
    for heads in (0, 5, -1):
        with pytest.raises(RuntimeError):
            slot.slot_rows(heads)


def _token(device, heads, seed):
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.nn.functional.normalize(torch.randn((1, 1, heads // 2, 128), generator=gen),
                                          dim=-1).bfloat16() for _ in range(2))
    v = torch.randn((1, 1, heads, 128), generator=gen).bfloat16()
    g = -0.1 * torch.rand((1, 1, heads), generator=gen)
    b = torch.sigmoid(torch.randn((1, 1, heads), generator=gen)).bfloat16()
    return [t.to(device) for t in (q, k, v, g, b)]


def test_runtime_fork(device):
    """A fork goes on from where its source stands, through a refit, and each on its own."""
    heads = 4
    runtime = gdn.GdnStateCodecRuntime()
    state = 0.1 * filled((5, heads, 128, 128), torch.float32, device)
    tokens = [_token(device, heads, i) for i in range(24)]

    def step(index, token):
        return runtime.step(state, index, *token, 128 ** -0.5).clone()

    with pytest.raises(RuntimeError, match="no slot"):
        runtime.fork(1, [2])
    step(1, tokens[0])
    with pytest.raises(RuntimeError, match="negative"):
        runtime.fork(1, [2, -1])
    assert list(runtime._slots) == [1]
    runtime.invalidate([1])
    for token in tokens[:9]:
        step(1, token)
    step(4, tokens[0])  # a slot of its own, forgotten by the fork
    runtime.fork(1, [3, 4, 4, 1])
    live = runtime._slots[1].window
    for index in (3, 4):
        other = runtime._slots[index].window
        for a, b in zip(live.slot_rows(heads), other.slot_rows(heads)):
            assert torch.equal(bits(a), bits(b)) and a.data_ptr() != b.data_ptr()
    step(3, tokens[20])  # a token of its own changes no other
    for token in tokens[9:20]:
        assert torch.equal(step(1, token), step(4, token))
    assert not torch.equal(step(3, tokens[9]), step(1, tokens[9]))
    runtime.fork(1, [])
    runtime.close()


# ---------------------------------------------------------------- refusals

def test_refusals(device):
    s, t = ints([0, 1], device), ints([2, 3], device)
    moves = gdn.slot_moves(s, t, 4)
    for bad in ((s[:1], t, 4), (s.long(), t, 4), (s, t.cpu(), 4), (s, t, 0), (s, t, 2 ** 31),
                (s, t, -1), (ints([], device), ints([], device), 4),
                (ints([0] * 4097, device), ints([0] * 4097, device), 9),
                (s.view(1, 2), t.view(1, 2), 4)):
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            gdn.slot_moves(*bad)
    for bad in (s.long(), s.bool(), s.cpu(), ints([], device), ints([1] * 65537, device),
                s.view(1, 2)):
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            gdn.compaction_moves(bad)
    x = torch.ones((4, 8), device=device)
    before = x.clone()
    wide = torch.ones((4, 16), device=device)
    long = torch.ones((7, 8), device=device)
    for bad in (([], moves), (x[:3], moves), (torch.ones((5, 8), device=device), moves),
                (wide[:, :8], moves), (x.t(), moves), (x.cpu(), moves),
                ([x, x], moves), ([x, x.view(4, 4, 2)], moves), ([long[:4], long[3:]], moves),
                (torch.tensor(1.0, device=device), moves),
                (x, moves._replace(steps=moves.steps.long())),
                (x, moves._replace(steps=moves.steps[:0])),
                (x, moves._replace(steps=moves.steps[:, :2])),
                (x, moves._replace(steps=moves.steps.cpu())),
                (x, moves._replace(steps=moves.steps[0])),
                (x.clone().requires_grad_(), moves),
                (x, moves, [x.clone(), x.clone()]), (x, moves, x), (x, moves, wide),
                (x, moves, x.clone().bfloat16()), (x, moves, x.cpu()),
                ([x, wide], moves, [long[:4], long[3:].repeat(1, 2)[:, :16].clone()[:3]]),
                ([x, x], moves, [wide.view(8, 8)[:4], wide.view(8, 8)[2:6]]),
                (long[:4], moves, long[3:]),
                # read from one address: the longer of the two overlaps what is written
                ([wide.view(-1)[:64].view(4, 16), wide.view(-1)[:16].view(4, 4)], moves,
                 [wide.clone(), wide.view(-1)[48:].view(4, 4)]),
                ([wide, wide], moves, [wide.clone(), wide])):
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            gdn.copy_slots(*bad)
    assert torch.equal(x, before)
