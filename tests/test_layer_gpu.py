"""The layer operators on the GPU against float64 (tests/delta_reference.py).

Tolerances, from the arithmetic.  A bf16 output is held to the float64 value
rounded to bf16 (whose own rounding, up to 2^-8 of a value, would hide more): the two
differ, by one step of 2^-7 at most, only where the exact value is so near the middle
between two that the kernel's 2^-15 decides.  2^-9 + 2^-12 in the 2-norm leaves room
for a tenth of the values to do so.  An fp32 state or gradient is a chain of some
hundred fp32 additions a chunk, of terms that are rounded once or twice (2^-24 each):
with the roundings independent about 20 x 2^-24 = 2^-19.7, and 2^-18 leaves a factor
of 3 for what the solve amplifies (keys here are random unit vectors; where they are
all alike, 2^-16).  A log decay's gradient is a sum of differences of such numbers,
some ten times larger than it: 2^-15."""

from __future__ import annotations

import pytest
import torch

import delta_reference as ref
import gdn_state_codec as gdn
from gdn_state_codec import layer

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -9 + 2.0 ** -12
FP32 = 2.0 ** -18
DECAY = 2.0 ** -15


def close(got, want, bound, name=""):
    rounded = want.to(got.dtype) if got.dtype == torch.bfloat16 else want
    got, want = got.detach().double().cpu(), rounded.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), name
    off, size = float((got - want).norm()), float(want.norm())
    print(f"{name}: {off / size if size else off:.3g} (bound {bound:.3g})", flush=True)
    assert off <= bound * size + 1e-30, (name, off, size)


def tokens_of(total, heads, key_heads, seed, decay="mixed", alike=False):
    """One fused projection's slices on the CPU: q, k, v (bf16), log decay, beta."""
    gen = torch.Generator().manual_seed(seed)
    mixed = torch.randn((total, (2 * key_heads + heads) * 128), generator=gen).bfloat16()
    if alike:
        mixed[:, key_heads * 128:2 * key_heads * 128] = mixed[:1, :key_heads * 128]
    q = mixed[:, :key_heads * 128].view(total, key_heads, 128)
    k = mixed[:, key_heads * 128:2 * key_heads * 128].view(total, key_heads, 128)
    v = mixed[:, 2 * key_heads * 128:].view(total, heads, 128)
    rate = {"mixed": torch.exp(-6.0 + 6.0 * torch.rand((1, heads), generator=gen)),
            "none": torch.zeros(1, heads), "strong": torch.full((1, heads), 20.0)}[decay]
    log_decay = -rate * torch.rand((total, heads), generator=gen)
    beta = torch.sigmoid(torch.randn((total, heads), generator=gen)).bfloat16()
    return mixed, q, k, v, log_decay, beta


def on(device, mixed, q, k, v, log_decay, beta):
    """The same on the GPU, q, k and v slices of one tensor there too."""
    m = mixed.to(device)
    a, b = q.shape[1] * 128, 2 * q.shape[1] * 128
    return (m[:, :a].view(q.shape), m[:, a:b].view(k.shape), m[:, b:].view(v.shape),
            log_decay.to(device), beta.to(device))


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


# ------------------------------------------------------------------- tables

@pytest.mark.parametrize("lengths,most", [
    ([1], 1), ([0], 0), ([64], 64), ([65, 0, 1, 63, 64, 128, 129], 600), ([5, -3, 7], 100),
    ([100, 200, 300], 250), ([100, 200, 300], 0), ([2 ** 31 - 1, 2 ** 31 - 1, 5], 1000),
    (list(range(300)), 50000), ([3] * 4096, 20000), ([0] * 4000 + [700] * 96, 70000)])
def test_request_tables(device, lengths, most):
    slots = [(7 * i) % 9001 - 1 for i in range(len(lengths))]
    t = gdn.request_tables(ints(lengths, device), ints(slots, device), most)
    rows = layer.table_rows(most, len(lengths))
    for got, want in zip(t, ref.tables(lengths, slots, most, rows)):
        want = torch.tensor(want, dtype=torch.int32)
        assert got.dtype == torch.int32 and got.is_contiguous() and got.data_ptr() % 16 == 0
        assert torch.equal(got.cpu(), want.reshape(got.shape))


# --------------------------------------------------------------- one token

@pytest.mark.parametrize("batch,heads,key_heads,pool_dtype,normalize", [
    (1, 1, 1, torch.float32, True), (3, 4, 2, torch.float32, False),
    (7, 6, 2, torch.bfloat16, True), (40, 32, 16, torch.float32, True),
    (33, 32, 32, torch.bfloat16, False), (5, 8, 1, torch.float32, True)])
def test_step(device, batch, heads, key_heads, pool_dtype, normalize):
    x = tokens_of(batch, heads, key_heads, 11)
    scale = 0.25 if not normalize else layer.QUERY_SCALE
    gen = torch.Generator().manual_seed(12)
    pool = (0.1 * torch.randn((batch + 4, heads, 128, 128), generator=gen)).to(pool_dtype)
    slots = torch.randperm(batch + 4, generator=gen)[:batch].int()
    if batch > 2:
        slots[1] = -1
    if batch > 3:
        slots[2] = batch + 4  # outside the pool: skipped too
    live = ((slots >= 0) & (slots < batch + 4)).nonzero()[:, 0]
    q, k, v, g, b = on(device, *x)
    if not normalize:
        k = (k * 0.1).contiguous()
        x = (*x[:2], (x[2] * 0.1), *x[3:])
    dev = pool.to(device)
    out = torch.full((batch, heads, 128), 3.0, dtype=torch.bfloat16, device=device)
    got = gdn.gated_delta_step(q, k, v, g, b, dev, slots.to(device), scale=scale,
                               normalize=normalize, out=out)
    assert got is out
    want, final = ref.rule(*(t[live] for t in x[1:]), [1] * len(live), pool[slots[live].long()],
                           scale, normalize)
    close(out[live.to(device)], want, BF16, "out")
    close(dev[slots[live].long().to(device)], final,
          FP32 if pool_dtype == torch.float32 else BF16, "states")
    rest = torch.ones(batch + 4, dtype=torch.bool)
    rest[slots[live].long()] = False
    assert torch.equal(dev.cpu()[rest], pool[rest])  # other slots are untouched
    dead = torch.ones(batch, dtype=torch.bool)
    dead[live] = False
    assert (out.cpu()[dead] == 3.0).all()


def test_step_matches_prefill_of_one_token(device):
    x = on(device, *tokens_of(6, 4, 2, 13))
    pool = torch.randn((6, 4, 128, 128), device=device) * 0.1
    slots = ints([4, 0, 5, 2, 1, 3], device)
    other = pool.clone()
    a = gdn.gated_delta_step(*x, pool, slots)
    t = gdn.request_tables(ints([1] * 6, device), slots, 6)
    b = gdn.gated_delta_prefill(*x, t, slots, other)
    close(a, b.cpu(), BF16, "out")
    close(pool, other.cpu(), FP32, "states")


# ----------------------------------------------------------------- prefill

LENGTHS = [[1], [64], [65], [0, 1, 63, 64, 65, 130, 0], [257, 2], [0], [127, 128, 129]]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("heads,key_heads,pool_dtype,normalize", [
    (1, 1, torch.float32, True), (4, 2, torch.bfloat16, True), (3, 1, torch.float32, False),
    (8, 8, torch.float32, True)])
def test_prefill(device, lengths, heads, key_heads, pool_dtype, normalize):
    _prefill(device, lengths, heads, key_heads, pool_dtype, normalize, seed=21)


@pytest.mark.parametrize("decay", ["none", "strong"])
def test_prefill_decays(device, decay):
    _prefill(device, [130, 5, 64], 4, 2, torch.float32, True, seed=22, decay=decay)


def test_prefill_of_keys_that_are_all_alike(device):
    """A_ij is then close to 1 everywhere: the solve's worst case."""
    _prefill(device, [200], 2, 1, torch.float32, True, seed=23, decay="none", alike=True,
             state_bound=2.0 ** -16)


def test_prefill_of_many_heads_takes_the_wide_form(device):
    """More than 32 requests x heads: whole heads a workgroup."""
    _prefill(device, [100, 30, 0, 64, 129, 1, 70, 3, 65], 6, 3, torch.float32, True, seed=24)


@pytest.mark.parametrize("pool_dtype,normalize", [
    (torch.bfloat16, True), (torch.float32, False)])
@pytest.mark.parametrize("lengths", [[1] * 9, [64] * 9, [0, 330, 2, 63, 65, 0, 128, 127, 5]])
def test_prefill_variants_of_the_wide_form(device, lengths, pool_dtype, normalize):
    _prefill(device, lengths, 4, 2, pool_dtype, normalize, seed=27)


@pytest.mark.parametrize("lengths,heads,key_heads,pool_dtype,normalize,decay", [
    ([4160], 2, 1, torch.float32, True, "mixed"),
    ([4100], 1, 1, torch.bfloat16, True, "none"),
    ([5003], 3, 3, torch.float32, False, "mixed"),
    ([9000, 3, 0, 7500], 2, 2, torch.float32, True, "mixed"),
    ([4096, 4300], 8, 4, torch.bfloat16, True, "strong"),
    ([8300], 32, 16, torch.float32, True, "mixed"),
    ([70, 8200], 1, 1, torch.float32, True, "none")])
def test_prefill_of_long_sequences_in_segments(device, lengths, heads, key_heads, pool_dtype,
                                               normalize, decay):
    """64 chunks a request and more, and 4 for each of at most 32 requests x heads.  Many
    times the chunks of the other tests, but a state forgets (through its decays or its
    writes) what the first of them rounded."""
    _prefill(device, lengths, heads, key_heads, pool_dtype, normalize, seed=29, decay=decay)


def test_prefill_of_a_short_batch_in_a_long_buffer(device):
    """Segments by the buffer's length; the requests fill a few chunks of it."""
    lengths, slots = [130, 0, 64], ints([2, 1, 0], device)
    total, room = sum(lengths), 64 * 200
    mixed, q, k, v, g, b = tokens_of(room, 2, 1, 33)
    inputs = on(device, mixed, q, k, v, g, b)
    pool = torch.zeros((3, 2, 128, 128), device=device)
    tables = gdn.request_tables(ints(lengths, device), slots, room)
    out = gdn.gated_delta_prefill(*inputs, tables, slots, pool)
    want, final = ref.rule(*(t[:total] for t in (q, k, v, g, b)), lengths,
                           torch.zeros((3, 2, 128, 128), dtype=torch.float64))
    close(out[:total], want, BF16, "out")
    close(pool[slots.long()], final, FP32, "states")


def test_segments_skip_padding_and_forget_and_replay(device):
    """A padding request among long ones, log decays of -inf at the segments' borders and
    inside, NaN in the padding's tokens, and a captured call's replays."""
    lengths, slots = [4200, 4300, 4160], ints([2, -1, 0], device)
    total, keep = sum(lengths), torch.cat([torch.arange(4200), torch.arange(8500, 12660)])
    mixed, q, k, v, g, b = tokens_of(total, 2, 1, 35, decay="none")
    for at in (0, 63, 64, 700, 8500, 12659):
        g[at] = float("-inf")
    g[1000:1100, 1] = -3.0e38
    mixed[4200:8500] = float("nan")
    start = 0.1 * torch.randn((3, 2, 128, 128), generator=torch.Generator().manual_seed(36))
    x = on(device, mixed, q, k, v, g, b)
    pool = start.to(device)
    out = torch.full((total, 2, 128), 7.0, dtype=torch.bfloat16, device=device)
    space = torch.empty(layer.workspace_bytes(total, 3, 2, 1), dtype=torch.uint8, device=device)
    tables = gdn.request_tables(ints(lengths, device), slots, total)

    def work():
        gdn.gated_delta_prefill(*x, tables, slots, pool, workspace=space, out=out)

    work()
    want, final = ref.rule(q[keep], k[keep], v[keep], g[keep], b[keep], [4200, 4160],
                           start[torch.tensor([2, 0])])
    close(out.cpu()[keep], want, BF16, "out")
    close(pool[[2, 0]], final, FP32, "states")
    assert (out[4200:8500].cpu() == 7.0).all() and torch.equal(pool[1].cpu(), start[1])
    eager = [out.clone(), pool.clone()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for _ in range(3):
        pool.copy_(start)
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(pool, eager[1])


def _prefill(device, lengths, heads, key_heads, pool_dtype, normalize, seed, decay="mixed",
             alike=False, state_bound=FP32):
    n, total = len(lengths), sum(lengths)
    rest = 5  # rows of no request: NaN there must not reach anything
    x = tokens_of(total + rest, heads, key_heads, seed, decay, alike)
    if not normalize:
        x[0][:, key_heads * 128:2 * key_heads * 128] *= 0.1  # k is a slice of it
    for t in (x[0], x[4], x[5]):
        t[total:] = float("nan")
    gen = torch.Generator().manual_seed(seed + 1)
    pool = (0.1 * torch.randn((n + 2, heads, 128, 128), generator=gen)).to(pool_dtype)
    slots = torch.randperm(n + 2, generator=gen)[:n].int()
    resume = torch.tensor([i % 3 != 1 for i in range(n)], dtype=torch.int32)
    scale = layer.QUERY_SCALE if normalize else 0.5
    inputs = on(device, *x)
    dev = pool.to(device)
    tables = gdn.request_tables(ints(lengths, device), slots.to(device), total + rest)
    out = torch.full((total + rest, heads, 128), 7.0, dtype=torch.bfloat16, device=device)
    got = gdn.gated_delta_prefill(*inputs, tables, slots.to(device), dev,
                                  resume=resume.to(device), scale=scale, normalize=normalize,
                                  out=out)
    assert got is out
    initial = pool[slots.long()].double() * resume[:, None, None, None]
    want, final = ref.rule(*(t[:total] for t in x[1:]), lengths, initial, scale, normalize)
    if total:
        close(out[:total], want, BF16 if not alike else 2 * BF16, "out")
    assert (out[total:].cpu() == 7.0).all()
    close(dev[slots.long().to(device)], final,
          state_bound if pool_dtype == torch.float32 else BF16, "states")
    other = torch.ones(n + 2, dtype=torch.bool)
    other[slots.long()] = False
    assert torch.equal(dev.cpu()[other], pool[other])


def test_prefill_skips_padding(device):
    lengths, slots = [70, 30, 66], ints([2, -1, 0], device)
    mixed, q, k, v, g, b = tokens_of(166, 2, 2, 31)
    mixed[70:100] = float("nan")
    pool = 0.1 * torch.randn((3, 2, 128, 128), generator=torch.Generator().manual_seed(32))
    dev = pool.to(device)
    out = torch.full((166, 2, 128), 7.0, dtype=torch.bfloat16, device=device)
    tables = gdn.request_tables(ints(lengths, device), slots, 166)
    gdn.gated_delta_prefill(*on(device, mixed, q, k, v, g, b), tables, slots, dev, out=out)
    keep = torch.cat([torch.arange(70), torch.arange(100, 166)])
    want, final = ref.rule(q[keep], k[keep], v[keep], g[keep], b[keep], [70, 66],
                           pool[torch.tensor([2, 0])])
    close(out.cpu()[keep], want, BF16, "out")
    close(dev[[2, 0]], final, FP32, "states")
    assert (out[70:100].cpu() == 7.0).all() and torch.equal(dev[1].cpu(), pool[1])


def test_prefill_in_pieces_is_prefill_at_once(device):
    """300 tokens in one call, or 100, 7 and 193 resumed from the pool."""
    x = on(device, *tokens_of(300, 4, 2, 33))
    whole, pieces = (torch.zeros((1, 4, 128, 128), device=device) for _ in range(2))
    slot, outs = ints([0], device), []
    fresh, go_on = ints([0], device), ints([1], device)
    one = gdn.gated_delta_prefill(
        *x, gdn.request_tables(ints([300], device), slot, 300), slot, whole, resume=fresh)
    for begin, end in ((0, 100), (100, 107), (107, 300)):
        part = [t[begin:end] for t in x]
        part[3:] = [t.contiguous() for t in part[3:]]
        tables = gdn.request_tables(ints([end - begin], device), slot, end - begin)
        outs.append(gdn.gated_delta_prefill(*part, tables, slot, pieces,
                                            resume=fresh if begin == 0 else go_on))
    close(torch.cat(outs), one.double().cpu(), BF16, "out")
    close(pieces, whole.double().cpu(), FP32, "state")


def test_log_decay_of_minus_infinity_forgets(device):
    mixed, q, k, v, g, b = tokens_of(100, 2, 1, 34)
    g[40] = float("-inf")
    g[63] = float("-inf")
    g[64, 1] = -3.0e38
    pool = torch.ones((1, 2, 128, 128), device=device)
    slot = ints([0], device)
    out = gdn.gated_delta_prefill(*on(device, mixed, q, k, v, g, b),
                                  gdn.request_tables(ints([100], device), slot, 100), slot, pool)
    want, final = ref.rule(q, k, v, g, b, [100], torch.ones(1, 2, 128, 128))
    close(out, want, BF16, "out")
    close(pool, final, FP32, "state")


def test_states_past_four_gibibytes(device):
    """A slot and a token row whose byte offsets pass 2^32."""
    pool = torch.empty((4600, 16, 128, 128), device=device)  # 4.8 GB
    slot = ints([4599], device)
    pool[4599] = 0.05
    mixed, q, k, v, g, b = tokens_of(3, 16, 16, 35)
    step = (1 << 24) - 8  # elements between tokens: the largest allowed, times 200
    far = torch.empty((200 * step + 6144,), dtype=torch.bfloat16, device=device)
    rows = far.as_strided((200, 6144), (step, 1))
    rows[197:] = mixed.to(device)
    parts = [rows[:, 2048 * i:2048 * (i + 1)].unflatten(1, (16, 128)) for i in range(3)]
    g_all, b_all = torch.zeros((200, 16)), torch.zeros((200, 16)).bfloat16()
    g_all[197:], b_all[197:] = g, b
    rows[:197] = 0.0
    tables = gdn.request_tables(ints([200], device), slot, 200)
    out = gdn.gated_delta_prefill(*parts, g_all.to(device), b_all.to(device), tables, slot, pool)
    want, final = ref.rule(q, k, v, g, b, [3], torch.full((1, 16, 128, 128), 0.05))
    close(out[197:], want, BF16, "out")
    close(pool[4599:], final, FP32, "state")
    token = [p[199:200] for p in parts]
    before = pool[4599:].double().cpu()
    out = gdn.gated_delta_step(*token, g[2:].contiguous().to(device), b[2:].contiguous().to(device),
                               pool, slot)
    want, final = ref.rule(q[2:], k[2:], v[2:], g[2:], b[2:], [1], before)
    close(out, want, BF16, "step out")
    close(pool[4599:], final, FP32, "step state")


def test_side_stream_and_graph_replays(device):
    """Calls go to the current stream, and a captured prefill and step replay."""
    lengths = [70, 5]
    x = on(device, *tokens_of(75, 4, 2, 36))
    slots = ints([1, 0], device)
    pool = torch.zeros((2, 4, 128, 128), device=device)
    out = torch.zeros((75, 4, 128), dtype=torch.bfloat16, device=device)
    size = layer.workspace_bytes(75, 2, 4, 2)
    space = torch.empty(size, dtype=torch.uint8, device=device)
    lens = ints(lengths, device)
    last = [t[[69, 74]].contiguous() for t in x]
    stepped = torch.zeros((2, 4, 128), dtype=torch.bfloat16, device=device)

    def work():
        tables = gdn.request_tables(lens, slots, 75)
        gdn.gated_delta_prefill(*x, tables, slots, pool, workspace=space, out=out)
        gdn.gated_delta_step(*last, pool, slots, out=stepped)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    stream.synchronize()
    eager = [t.clone() for t in (out, stepped, pool)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for _ in range(3):
        pool.zero_()
        out.zero_()
        stepped.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((out, stepped, pool), eager):
            assert torch.equal(got, want)


# ---------------------------------------------------------------- training

TRAINED = ("queries", "keys", "values", "log_decay", "beta", "initial")


def _train(device, lengths, heads, key_heads, seed, scale=layer.QUERY_SCALE, normalize=True,
           decay="mixed", resumed=True, final_used=True, rest=0):
    n, total = len(lengths), sum(lengths)
    x = tokens_of(total + rest, heads, key_heads, seed, decay)
    if not normalize:
        x[0][:, key_heads * 128:2 * key_heads * 128] *= 0.1
    gen = torch.Generator().manual_seed(seed + 1)
    initial = 0.1 * torch.randn((n, heads, 128, 128), generator=gen)
    d_out = torch.randn((total + rest, heads, 128), generator=gen).bfloat16()
    d_final = 0.1 * torch.randn((n, heads, 128, 128), generator=gen)
    if not resumed:
        initial.zero_()
    if not final_used:
        d_final.zero_()
    for t in (x[0], x[4], x[5], d_out):
        t[total:] = float("nan")
    leaves = [t.detach().requires_grad_(True) for t in on(device, *x)]
    start = initial.to(device).requires_grad_(True) if resumed else None
    slots = ints(list(range(n)), device)
    tables = gdn.request_tables(ints(lengths, device), slots, total + rest)
    out, final = gdn.gated_delta_rule(*leaves, tables, start, scale, normalize)
    wanted = leaves + ([start] if resumed else [])
    outs = [out, final] if final_used else [out]
    given = [d_out.to(device), d_final.to(device)][:len(outs)]
    grads = torch.autograd.grad(outs, wanted, given)
    cut = [t[:total] for t in x[1:]]
    want_out, want_final = ref.rule(*cut, lengths, initial, scale, normalize)
    want = ref.rule_gradients(*cut, lengths, initial, d_out[:total], d_final, scale, normalize)
    if total:
        close(out[:total], want_out, BF16, "out")
    close(final, want_final, FP32, "final")
    for name, got, expected in zip(TRAINED, grads, want):
        bound = {"log_decay": DECAY, "initial": FP32}.get(name, BF16)
        if name != "initial":
            assert (got[total:] == 0).all(), name  # tokens of no request
            got = got[:total]
        if got.numel():
            close(got, expected, bound, f"d_{name}")
    assert (out[total:] == 0).all()


@pytest.mark.parametrize("lengths", [[1], [64], [65, 3], [0, 1, 63, 130, 0], [200]])
@pytest.mark.parametrize("heads,key_heads", [(1, 1), (4, 2), (3, 1), (4, 1)])
def test_train(device, lengths, heads, key_heads):
    _train(device, lengths, heads, key_heads, 41)


@pytest.mark.parametrize("options", [
    dict(normalize=False, scale=0.5), dict(decay="none"), dict(decay="strong"),
    dict(resumed=False), dict(final_used=False), dict(rest=70), dict(resumed=False, rest=3)])
def test_train_variants(device, options):
    _train(device, [70, 0, 129], 4, 2, 43, **options)


def test_train_of_many_heads_takes_the_wide_form(device):
    _train(device, [65, 20, 0, 70, 1], 8, 4, 45)


@pytest.mark.parametrize("options", [
    dict(), dict(normalize=False, scale=0.5), dict(decay="none"), dict(decay="strong"),
    dict(resumed=False), dict(final_used=False), dict(rest=700)])
def test_train_variants_of_the_wide_form(device, options):
    _train(device, [200, 1, 64, 0, 130, 63], 6, 3, 47, **options)


def test_train_of_one_chunk_and_of_many_in_both_forms(device):
    _train(device, [330], 2, 1, 49)
    _train(device, [330] + [2] * 16, 2, 1, 51)


def test_forward_differences_of_the_kernels_themselves(device):
    """<d_log_decay, way> and <d_initial, way> against differences of the kernels' own
    fp32 final states.  A decay's step runs through up to 150 tokens' product, h
    sqrt(150) = 0.25 at h = 0.02, whose square is too much for a central difference
    to ignore; with the points at 2 h the quotient is off by its fourth power over 30
    and by 2^-20 |value terms| / h: 1e-3."""
    lengths, heads = [150], 2
    x = tokens_of(150, heads, 1, 47)
    q, k, v, g, b = on(device, *x)
    gen = torch.Generator().manual_seed(48)
    weight = torch.randn((1, heads, 128, 128), generator=gen).to(device)
    start = (0.1 * torch.randn((1, heads, 128, 128), generator=gen)).to(device)
    tables = gdn.request_tables(ints(lengths, device), ints([0], device), 150)
    leaves = [g.clone().requires_grad_(True), start.clone().requires_grad_(True)]
    _, final = gdn.gated_delta_rule(q, k, v, leaves[0], b, tables, leaves[1])
    grads = torch.autograd.grad([final], leaves, [weight])

    def value(g, s):
        with torch.no_grad():
            return float((gdn.gated_delta_rule(q, k, v, g, b, tables, s)[1].double()
                          * weight).sum())

    for i, h in ((0, 0.02), (1, 0.02)):
        way = torch.randn(leaves[i].shape, generator=gen).to(device)
        at = []
        for steps in (-2, -1, 1, 2):
            moved = [g, start]
            moved[i] = moved[i] + steps * h * way
            at.append(value(*moved))
        slope = (8 * (at[2] - at[1]) - (at[3] - at[0])) / (12 * h)
        want = float((grads[i].double() * way).sum())
        size = float(grads[i].double().norm())
        print(f"differences {i}: {slope} {want} {size}", flush=True)
        assert abs(slope - want) <= 1e-3 * max(abs(want), size)


def test_backward_twice_gives_the_same(device):
    x = [t.detach().requires_grad_(True) for t in on(device, *tokens_of(130, 4, 2, 49))]
    tables = gdn.request_tables(ints([130], device), ints([0], device), 130)
    out, final = gdn.gated_delta_rule(*x, tables)
    d = torch.randn_like(out)
    first = torch.autograd.grad([out], x, [d], retain_graph=True)
    second = torch.autograd.grad([out], x, [d])
    for a, b in zip(first, second):
        assert torch.equal(a, b)


# ------------------------------------------------------------------- norms

def _norm_bound(dtype):
    return BF16 if dtype == torch.bfloat16 else FP32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 128), (3, 1, 128), (5, 7, 128), (1030, 2, 128)])
def test_gated_norm(device, dtype, shape):
    gen = torch.Generator().manual_seed(51)
    x = (3.0 * torch.randn(shape, generator=gen)).to(dtype)
    gate = (4.0 * torch.randn(shape, generator=gen)).to(dtype)
    weight = 1.0 + 0.2 * torch.randn(128, generator=gen)
    d = torch.randn(shape, generator=gen).to(dtype)
    x.view(-1, 128)[0] = 0.0  # a row of zeros
    leaves = [t.to(device).requires_grad_(True) for t in (x, gate, weight)]
    out = gdn.gated_norm(*leaves, eps=1e-4)
    with torch.no_grad():
        assert torch.equal(gdn.gated_norm(*leaves, eps=1e-4), out)
    close(out, ref.norm(x, weight, ref.silu(gate), 1e-4), _norm_bound(dtype), "out")
    d_x, d_gate, d_weight = torch.autograd.grad([out], leaves, [d.to(device)])
    want, terms, d_through = ref.norm_gradients(x, weight, ref.silu(gate), d, 1e-4)
    close(d_x, want, _norm_bound(dtype), "d_x")
    close(d_gate, d_through * ref.silu_slope(gate), _norm_bound(dtype), "d_gate")
    off = (d_weight.double().cpu() - terms.sum(0)).abs()
    assert (off <= FP32 * terms.abs().sum(0) + 1e-30).all()


@pytest.mark.parametrize("dtype,stream", [
    (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
    (torch.float32, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("rows,width", [
    (1, 8), (3, 64), (1, 512), (9, 520), (5, 1024), (6, 1032), (2, 2048), (5, 4096), (3, 4104),
    (2, 8200), (1, 16384), (2100, 128), (2100, 1536)])
def test_residual_norm(device, dtype, stream, rows, width):
    gen = torch.Generator().manual_seed(53)
    x = torch.randn((rows, width), generator=gen).to(dtype)
    residual = (2.0 * torch.randn((rows, width), generator=gen)).to(stream)
    weight = 1.0 + 0.2 * torch.randn(width, generator=gen)
    d = torch.randn((rows, width), generator=gen).to(dtype)
    d_sum = torch.randn((rows, width), generator=gen).to(stream)
    leaves = [t.to(device).requires_grad_(True) for t in (x, residual, weight)]
    out, total = gdn.residual_norm(*leaves, scale=0.75, eps=1e-5)
    with torch.no_grad():
        again = gdn.residual_norm(*leaves, scale=0.75, eps=1e-5)
        assert torch.equal(again[0], out) and torch.equal(again[1], total)
    exact = residual.double() + 0.75 * x.double()
    close(total, exact, _norm_bound(stream), "sum")
    stored = total.detach().cpu()  # the norm is of what the stream holds
    close(out, ref.norm(stored, weight, 1.0, 1e-5), _norm_bound(dtype), "out")
    for given in (d_sum, None):
        outs, ds = ([out, total], [d, d_sum]) if given is not None else ([out], [d])
        d_x, d_residual, d_weight = torch.autograd.grad(
            outs, leaves, [t.to(device) for t in ds], retain_graph=True)
        want, terms, _ = ref.norm_gradients(stored, weight, 1.0, d, 1e-5)
        if given is not None:
            want = want + d_sum.double()
        close(d_residual, want, _norm_bound(stream), "d_residual")
        close(d_x, 0.75 * want, _norm_bound(dtype), "d_x")
        off = (d_weight.double().cpu() - terms.sum(0)).abs()
        assert (off <= FP32 * terms.abs().sum(0) + 1e-30).all()


def test_norm_rows_do_not_mix(device):
    """A NaN or an infinity stays in its own row."""
    x = torch.randn((40, 2048), device=device)
    clean = gdn.residual_norm(x, x, torch.ones(2048, device=device))[0]
    bad = x.clone()
    bad[3, 7], bad[20, 0] = float("nan"), float("inf")
    got = gdn.residual_norm(bad, bad, torch.ones(2048, device=device))[0]
    keep = [i for i in range(40) if i not in (3, 20)]
    assert torch.equal(got[keep], clean[keep]) and torch.isnan(got[3]).all()
    heads, gate = x.view(-1, 128), torch.randn((640, 128), device=device)
    weight = torch.ones(128, device=device)
    clean = gdn.gated_norm(heads, gate, weight)
    got = gdn.gated_norm(bad.view(-1, 128), gate, weight)
    keep = [i for i in range(640) if i not in (48, 320)]
    assert torch.equal(got[keep], clean[keep]) and torch.isnan(got[48]).all()


def test_norm_gradients_are_the_kernels_differences(device):
    """fp32 values, step 1e-2: the quotient is off by about 1e-4 of the slope and
    2^-22 |value| / 1e-2."""
    gen = torch.Generator().manual_seed(55)
    x, gate, d = (torch.randn((6, 128), generator=gen).to(device) for _ in range(3))
    weight = (1.0 + 0.2 * torch.randn(128, generator=gen)).to(device)
    leaves = [t.clone().requires_grad_(True) for t in (x, gate, weight)]
    grads = torch.autograd.grad([gdn.gated_norm(*leaves)], leaves, [d])
    for i in range(3):
        way = torch.randn(leaves[i].shape, generator=gen).to(device)
        up, down = [x, gate, weight], [x, gate, weight]
        up[i], down[i] = up[i] + 1e-2 * way, down[i] - 1e-2 * way
        value = lambda a: float((gdn.gated_norm(*a).double() * d).sum())  # noqa: E731
        slope, want = (value(up) - value(down)) / 2e-2, float((grads[i].double() * way).sum())
        assert abs(slope - want) <= 2e-3 * max(1.0, abs(want)), (i, slope, want)


def test_empty_batches(device):
    empty = torch.empty((0, 4, 128), dtype=torch.bfloat16, device=device)
    assert gdn.gated_norm(empty, empty, torch.ones(128, device=device)).shape == empty.shape
    wide = torch.empty((0, 256), device=device)
    out, total = gdn.residual_norm(wide, wide, torch.ones(256, device=device))
    assert out.shape == total.shape == wide.shape
    pool = torch.ones((2, 4, 128, 128), device=device)
    g, b = (torch.empty((0, 4), dtype=t, device=device) for t in (torch.float32, torch.bfloat16))
    out = gdn.gated_delta_step(empty[:, :2], empty[:, :2], empty, g, b, pool, ints([], device))
    assert out.shape == empty.shape and (pool == 1).all()


# ---------------------------------------------------------------- refusals

def _good(device):
    q, k, v, g, b = on(device, *tokens_of(10, 4, 2, 61))
    tables = gdn.request_tables(ints([6, 4], device), ints([1, 0], device), 10)
    return dict(queries=q, keys=k, values=v, log_decay=g, beta=b, tables=tables,
                slot_ids=ints([1, 0], device), pool=torch.zeros((3, 4, 128, 128), device=device))


def test_prefill_refusals(device):
    good = _good(device)
    gdn.gated_delta_prefill(**good)
    d, t = device, good["tables"]
    bad = [
        dict(queries=good["queries"].float()), dict(queries=good["queries"].cpu()),
        dict(queries=good["queries"][:9]), dict(keys=good["keys"][:, :1]),
        dict(values=good["values"][:, :3]), dict(values=good["values"][..., :64]),
        dict(values=good["values"].transpose(0, 1)), dict(keys=good["keys"].flip(-1)[..., ::2]),
        dict(log_decay=good["log_decay"].double()), dict(log_decay=good["log_decay"][:, :2]),
        dict(log_decay=good["log_decay"].t().contiguous().t()), dict(beta=good["beta"].float()),
        dict(tables=t._replace(chunks=t.chunks[:1])), dict(tables=t._replace(order=t.order[:1])),
        dict(tables=t._replace(offsets=t.offsets.long())), dict(slot_ids=ints([0], d)),
        dict(slot_ids=good["slot_ids"].long()), dict(pool=good["pool"].half()),
        dict(pool=good["pool"][:, :2]), dict(pool=good["pool"].transpose(2, 3)),
        dict(resume=ints([1], d)), dict(resume=torch.ones(2, dtype=torch.bool, device=d)),
        dict(out=torch.zeros((10, 4, 128), device=d)),
        dict(out=torch.zeros((9, 4, 128), dtype=torch.bfloat16, device=d)),
        dict(workspace=torch.empty(100, dtype=torch.uint8, device=d)),
        dict(workspace=torch.empty(1 << 24, dtype=torch.float32, device=d)),
    ]
    for change in bad:
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            gdn.gated_delta_prefill(**{**good, **change})
    # rows 4 elements apart from a 16-byte boundary
    odd = torch.zeros(10 * 516 + 4, dtype=torch.bfloat16, device=d)
    with pytest.raises(RuntimeError, match="GDN State Codec"):
        gdn.gated_delta_prefill(**{**good, "values": odd.as_strided((10, 4, 128), (516, 128, 1))})
    with pytest.raises(RuntimeError, match="launch failed: 1"):  # misaligned
        gdn.gated_delta_prefill(**{**good, "values": odd.as_strided((10, 4, 128), (512, 128, 1), 4)})


def test_other_refusals(device):
    good = _good(device)
    with pytest.raises(RuntimeError, match="GDN State Codec"):
        gdn.request_tables(ints([1], device), ints([1, 2], device), 4)
    with pytest.raises(RuntimeError, match="GDN State Codec"):
        gdn.request_tables(ints([1], device).long(), ints([1], device), 4)
    with pytest.raises(RuntimeError, match="GDN State Codec"):
        gdn.request_tables(ints([1], device), ints([1], device), -1)
    with pytest.raises(RuntimeError, match="GDN State Codec"):
        gdn.request_tables(ints([1] * 4097, device), ints([1] * 4097, device), 5000)
    five = [good[n] for n in ("queries", "keys", "values", "log_decay", "beta")]
    with pytest.raises(RuntimeError, match="GDN State Codec"):
        gdn.gated_delta_step(*five, good["pool"], good["slot_ids"])
    with pytest.raises(RuntimeError, match="GDN State Codec"):
        gdn.gated_delta_rule(*five, good["tables"], torch.zeros((1, 4, 128, 128), device=device))
    x = torch.zeros((2, 256), device=device)
    w = torch.ones(256, device=device)
    for args in ((x, x[:1], w), (x, x, w[:128]), (x.half(), x, w), (x, x.t(), w),
                 (x, x, w.bfloat16()), (x[:, ::2], x[:, ::2], w[:128]),
                 (x[:, :12].contiguous(), x[:, :12].contiguous(), w[:12].contiguous()),
                 (x.cpu(), x, w)):
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            gdn.residual_norm(*args)
    h, w = torch.zeros((3, 128), device=device), torch.ones(128, device=device)
    for args in ((h, h.bfloat16(), w), (h, h[:1], w), (h[:, :64], h[:, :64], w),
                 (h, h, w.double()), (x, x, w)):
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            gdn.gated_norm(*args)
