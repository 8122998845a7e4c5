"""Trees of drafted tokens on the state pool (gated_delta_tree, gated_delta_commit) on the
GPU against float64 (tests/draft_reference.py).

Tolerances, from the arithmetic.  An output is rounded to bf16 and is held to the float64
value rounded to bf16: as in tests/test_layer_gpu.py the two differ by a step of 2^-7 at
most, where the exact value lies near the middle of two, and 2^-9 + 2^-12 in the 2-norm
leaves room for a tenth of the values to do so.  A state is a sum of products of fp32
numbers along a path of up to 64 nodes: 2^-18 of its 2-norm, some 2^6 roundings of 2^-24,
as for a chunk of 64 tokens there."""

from __future__ import annotations

import pytest
import torch

import delta_reference as delta
import draft_reference as ref
import gdn_state_codec as gdn
from gdn_state_codec import layer

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -9 + 2.0 ** -12
FP32 = 2.0 ** -18
SHAPES = ("chain", "star", "branches", "roots", "any")


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def close(got, want, bound, name=""):
    rounded = want.to(got.dtype) if got.dtype == torch.bfloat16 else want
    got, want = got.detach().double().cpu(), rounded.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), name
    off, size = float((got - want).norm()), float(want.norm())
    print(f"{name}: {off / size if size else off:.3g} (bound {bound:.3g})", flush=True)
    assert off <= bound * size + 1e-30, (name, off, size)


def tokens_of(total, heads, key_heads, seed, decay="mixed", alike=False):
    """One fused projection on the CPU, and q, k, v (bf16, its slices), log decay, beta."""
    gen = torch.Generator().manual_seed(seed)
    mixed = torch.randn((total, (2 * key_heads + heads) * 128), generator=gen).bfloat16()
    if alike:
        mixed[:, key_heads * 128:2 * key_heads * 128] = mixed[:1, :key_heads * 128]
    rate = {"mixed": torch.exp(-6.0 + 6.0 * torch.rand((1, heads), generator=gen)),
            "none": torch.zeros(1, heads), "strong": torch.full((1, heads), 20.0)}[decay]
    log_decay = -rate * torch.rand((total, heads), generator=gen)
    beta = torch.sigmoid(torch.randn((total, heads), generator=gen)).bfloat16()
    return mixed, log_decay, beta


def parts(mixed, heads, key_heads):
    a, b = key_heads * 128, 2 * key_heads * 128
    rows = mixed.shape[0]
    return (mixed[:, :a].view(rows, key_heads, 128), mixed[:, a:b].view(rows, key_heads, 128),
            mixed[:, b:].view(rows, heads, 128))


class Batch:
    """Requests with trees, on both sides; slots in no order, the second padding and the
    third outside the pool where there are enough; rows of no request behind the last."""

    def __init__(self, device, shapes, heads, key_heads, pool_dtype, seed, normalize=True,
                 decay="mixed", alike=False, rest=3, padded=True):
        self.parents = [p for p in shapes]
        self.heads, self.key_heads, self.normalize = heads, key_heads, normalize
        self.scale = layer.QUERY_SCALE if normalize else 0.5
        n, self.total = len(shapes), sum(map(len, shapes))
        rows = self.total + rest
        self.mixed, self.g, self.b = tokens_of(rows, heads, key_heads, seed, decay, alike)
        if not normalize:
            self.mixed[:, key_heads * 128:2 * key_heads * 128] *= 0.1
        for t in (self.mixed, self.g, self.b):
            t[self.total:] = float("nan")
        gen = torch.Generator().manual_seed(seed + 1)
        self.pool = (0.1 * torch.randn((n + 2, heads, 128, 128), generator=gen)).to(pool_dtype)
        self.slots = torch.randperm(n + 2, generator=gen)[:n].int()
        if padded and n > 3:
            self.slots[1], self.slots[2] = -1, n + 2
        self.starts = [sum(map(len, shapes[:i])) for i in range(n)]
        self.device = device
        flat = [p for tree in shapes for p in tree] + [0] * rest
        self.dev_parents = ints(flat, device)
        self.dev_slots = self.slots.to(device)
        self.dev_mixed, self.dev_g, self.dev_b = (t.to(device)
                                                  for t in (self.mixed, self.g, self.b))
        self.dev_pool = self.pool.to(device)
        self.tables = gdn.request_tables(ints(list(map(len, shapes)), device), self.dev_slots,
                                         rows)

    def inputs(self):
        return (*parts(self.dev_mixed, self.heads, self.key_heads), self.dev_g, self.dev_b)

    def live(self):
        slots = self.pool.shape[0]
        return [r for r, slot in enumerate(self.slots.tolist()) if 0 <= slot < slots]

    def reference(self, r, nodes=None):
        """(out, states) of request r's first nodes."""
        tree = self.parents[r][:nodes]
        at = slice(self.starts[r], self.starts[r] + len(tree))
        q, k, v = parts(self.mixed, self.heads, self.key_heads)
        return ref.tree(q[at], k[at], v[at], self.g[at], self.b[at], tree,
                        self.pool[int(self.slots[r])], self.scale, self.normalize)

    def tree(self, out=None, **more):
        return gdn.gated_delta_tree(*self.inputs(), self.dev_parents, self.tables,
                                    self.dev_slots, self.dev_pool, scale=self.scale,
                                    normalize=self.normalize, out=out, **more)

    def commit(self, accepted):
        gdn.gated_delta_commit(*self.inputs()[1:], self.dev_parents,
                               ints(accepted, self.device), self.tables, self.dev_slots,
                               self.dev_pool, normalize=self.normalize)

    def check_tree(self, bound=BF16, max_nodes=64):
        out = torch.full((self.total + 3, self.heads, 128), 7.0, dtype=torch.bfloat16,
                         device=self.device)[:self.dev_mixed.shape[0]]
        assert self.tree(out, max_nodes=max_nodes) is out
        want = torch.full(out.shape, 7.0, dtype=torch.float64)
        for r in self.live():
            got, _ = self.reference(r, max_nodes)
            want[self.starts[r]:self.starts[r] + got.shape[0]] = got
        untouched = (want == 7.0).all(-1).all(-1)
        assert (out.cpu()[untouched] == 7.0).all()
        if not untouched.all():
            close(out.cpu()[~untouched], want[~untouched], bound, "out")
        assert torch.equal(self.dev_pool.cpu(), self.pool)  # the tree only reads it

    def check_commit(self, accepted, bound=None):
        self.dev_pool.copy_(self.pool)
        self.commit(accepted)
        want = self.pool.double()
        moved = []
        for r in self.live():
            if 0 <= accepted[r] < min(64, len(self.parents[r])):
                want[int(self.slots[r])] = self.reference(r)[1][accepted[r]]
                moved.append(int(self.slots[r]))
        got = self.dev_pool.cpu()
        rest = [i for i in range(self.pool.shape[0]) if i not in moved]
        assert torch.equal(got[rest], self.pool[rest])
        if moved:
            exact = self.pool.dtype == torch.float32
            close(got[moved], want[moved], bound or (FP32 if exact else BF16), "states")


FORMS = [(1, 1, torch.float32, True), (4, 2, torch.bfloat16, True),
         (3, 1, torch.float32, False), (8, 8, torch.float32, True),
         (5, 5, torch.bfloat16, False)]
SIZES = [[1], [5], [16], [17], [33], [64], [0, 1, 2, 15, 16, 17, 0], [31, 32, 33, 47, 48, 49],
         [63, 64, 64, 1]]


@pytest.mark.parametrize("heads,key_heads,pool_dtype,normalize", FORMS)
@pytest.mark.parametrize("sizes", SIZES)
def test_trees(device, sizes, heads, key_heads, pool_dtype, normalize):
    for i, shape in enumerate(SHAPES):
        batch = Batch(device, [ref.parents_of(shape, n, i) for n in sizes], heads, key_heads,
                      pool_dtype, 100 + i, normalize)
        print(shape, sizes, flush=True)
        batch.check_tree()


@pytest.mark.parametrize("heads,key_heads,pool_dtype,normalize", FORMS)
@pytest.mark.parametrize("sizes", SIZES)
def test_commits(device, sizes, heads, key_heads, pool_dtype, normalize):
    for i, shape in enumerate(SHAPES):
        batch = Batch(device, [ref.parents_of(shape, n, i) for n in sizes], heads, key_heads,
                      pool_dtype, 200 + i, normalize)
        print(shape, sizes, flush=True)
        batch.check_commit([n - 1 for n in sizes])
        batch.check_commit([(n // 2 if r % 2 else -1) for r, n in enumerate(sizes)])


@pytest.mark.parametrize("heads,key_heads", [(32, 16), (16, 16), (12, 3), (7, 7), (64, 16)])
@pytest.mark.parametrize("requests", [1, 9, 40])
def test_many_heads_and_requests(device, heads, key_heads, requests):
    """Grids of every size that a variant may be chosen by."""
    sizes = [(5 * i) % 19 for i in range(requests)]
    sizes[0] = 11
    batch = Batch(device, [ref.parents_of("any", n, 3) for n in sizes], heads, key_heads,
                  torch.float32, 31)
    batch.check_tree()
    batch.check_commit([n - 1 - r % 3 for r, n in enumerate(sizes)])


@pytest.mark.parametrize("max_nodes", [1, 2, 15, 16, 17, 32, 33, 63, 64])
def test_nodes_past_the_limit_are_left_as_they_were(device, max_nodes):
    batch = Batch(device, [ref.parents_of("any", n, 5) for n in (64, 20, 1, 0, 40, 70, 130)], 4,
                  2, torch.float32, 37, padded=False)
    batch.check_tree(max_nodes=max_nodes)


def test_requests_of_more_than_64_nodes(device):
    """Nodes from the 65th on are neither evaluated nor accepted."""
    batch = Batch(device, [ref.parents_of("chain", n) for n in (65, 200, 64, 3)], 2, 1,
                  torch.float32, 39, padded=False)
    batch.check_tree()
    batch.check_commit([64, 63, 63, 2])
    batch.check_commit([199, 64, 64, 3])


@pytest.mark.parametrize("decay", ["none", "strong"])
@pytest.mark.parametrize("shape", ["chain", "any"])
def test_decays(device, decay, shape):
    batch = Batch(device, [ref.parents_of(shape, n, 6) for n in (64, 30, 1, 17)], 4, 2,
                  torch.float32, 41, decay=decay, padded=False)
    batch.check_tree()
    batch.check_commit([63, 29, 0, 16])


@pytest.mark.parametrize("shape", ["chain", "any", "roots"])
def test_log_decays_of_minus_infinity_forget(device, shape):
    batch = Batch(device, [ref.parents_of(shape, n, 7) for n in (64, 20, 1)], 2, 1,
                  torch.float32, 43, padded=False)
    for at in (3, 15, 16, 40, 64, 70):
        batch.g[at] = float("-inf")
    batch.g[30, 1], batch.g[50, 0] = -3.0e38, -200.0
    batch.dev_g.copy_(batch.g)
    batch.check_tree()
    batch.check_commit([63, 19, 0])


@pytest.mark.parametrize("pool_dtype", [torch.float32, torch.bfloat16])
def test_log_decays_above_zero(device, pool_dtype):
    """States that grow, by up to e^32: the terms grow alike, so the bounds stay."""
    batch = Batch(device, [ref.parents_of(s, n, 9) for s, n in
                           (("chain", 64), ("any", 50), ("branches", 33), ("chain", 17))],
                  4, 2, pool_dtype, 47, padded=False)
    batch.g.uniform_(-0.3, 0.5, generator=torch.Generator().manual_seed(47))
    batch.g[:64, 0] = 0.5
    batch.dev_g.copy_(batch.g)
    batch.check_tree()
    batch.check_commit([63, 49, 32, 16])


def test_keys_that_are_all_alike(device):
    """Every write is over the same key: the solve's worst case, as in prefill's test."""
    batch = Batch(device, [ref.parents_of(s, 64, 8) for s in SHAPES], 2, 1, torch.float32, 45,
                  decay="none", alike=True, padded=False)
    batch.check_tree(2 * BF16)
    batch.check_commit([63] * 5, 2.0 ** -16)


def test_keys_of_zeros(device):
    """A row of zeros has no direction: nothing is read or written by it."""
    batch = Batch(device, [ref.parents_of("any", 20, 9)], 2, 1, torch.float32, 47)
    batch.mixed[4:9] = 0.0
    batch.dev_mixed.copy_(batch.mixed)
    batch.check_tree()
    batch.check_commit([19])


def test_parents_that_are_no_earlier_node(device):
    """Itself, a later node, one past the tree and any negative number are the cached
    state; no request's nodes are another's."""
    trees = [[-7, 0, 2, 9, 3, 2 ** 31 - 1, -2 ** 31, 64, 1], [5, 0, 1, 20, 3], [0, 1, 2, 3]]
    batch = Batch(device, trees, 4, 2, torch.float32, 49, padded=False)
    batch.check_tree()
    for accepted in ([8, 4, 3], [4, 2, 0]):
        batch.check_commit(accepted)


def test_one_slot_may_be_read_by_many_requests(device):
    batch = Batch(device, [ref.parents_of("any", n, 10) for n in (9, 30, 5, 9)], 2, 1,
                  torch.float32, 51, padded=False)
    batch.slots[:] = 1
    batch.dev_slots.fill_(1)
    batch.check_tree()


def test_accepted_places_that_are_no_node(device):
    batch = Batch(device, [ref.parents_of("chain", n) for n in (4, 4, 4, 4, 0, 4)], 2, 1,
                  torch.float32, 53, padded=False)
    batch.check_commit([4, -1, 2 ** 31 - 1, -2 ** 31, 0, 3])


def test_a_chain_is_the_step_token_by_token(device):
    """One tree call and one commit against gated_delta_step on the same pool."""
    batch = Batch(device, [ref.parents_of("chain", 20)], 4, 2, torch.float32, 55)
    out = batch.tree()
    stepped = batch.dev_pool.clone()
    outs = [gdn.gated_delta_step(*(t[i:i + 1] for t in batch.inputs()), stepped,
                                 batch.dev_slots) for i in range(20)]
    close(out[:20], torch.cat(outs).double().cpu(), BF16, "out")
    batch.commit([19])
    close(batch.dev_pool, stepped.double().cpu(), FP32, "states")


def test_outputs_whose_terms_cancel(device):
    """An output is good to 2^-18 of its terms (all fp32) and its own rounding of 2^-8,
    also where the cached state is 1,000 times the values."""
    batch = Batch(device, [ref.parents_of(s, 60, 11) for s in ("chain", "any")], 2, 1,
                  torch.float32, 57, decay="none", alike=True, padded=False, rest=0)
    batch.pool *= 1e4
    batch.b.fill_(1.0)
    batch.dev_pool.copy_(batch.pool)
    batch.dev_b.copy_(batch.b)
    out = batch.tree().double().cpu()
    q, k, v = parts(batch.mixed, 2, 1)
    unit, read = (delta.unit(x.double())[0] for x in (k[0, 0], q[:, 0]))
    for r in range(2):
        want, states = batch.reference(r)
        at = slice(batch.starts[r], batch.starts[r] + 60)
        # Writes are along one key: a write is as large as the state's reading of it and
        # the value, and 60 of them are summed.
        start = batch.pool[int(batch.slots[r])].double()
        terms = (torch.matmul(start.abs(), read[at].abs().t()).permute(2, 0, 1) * batch.scale
                 + batch.scale * (torch.matmul(start.abs(), unit.abs())[None]
                                  + 60 * v[at].double().abs().amax(0, keepdim=True)))
        bound = 2.0 ** -18 * terms + 2.0 ** -8 * want.abs()
        worst = float(((out[at] - want).abs() / bound).max())
        print(f"{worst:.3g}", flush=True)
        assert worst <= 1.0


def _below(parents, node):
    return [i for i in range(len(parents)) if node in ref.path(parents, i)]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("what", ["query", "key", "value", "decay", "strength"])
@pytest.mark.parametrize("nodes", [14, 40, 64])
def test_bad_values_stay_on_their_branch(device, nodes, what, bad):
    """Every other node's outputs are the very same, and every other request's."""
    trees = [ref.parents_of("any", nodes, 12), ref.parents_of("any", nodes, 13)]
    batch = Batch(device, trees, 4, 2, torch.float32, 59, padded=False, rest=0)
    clean = batch.tree().cpu()
    node = nodes // 4
    heads, columns = [0, 1], list(range(128))  # those of key head 0
    if what == "query":
        batch.dev_mixed[node, 5] = bad
        reached = [node]
    elif what == "key":
        batch.dev_mixed[node, 256 + 70] = bad
        reached = _below(trees[0], node)
    elif what == "value":
        batch.dev_mixed[node, 512 + 128 + 77] = bad
        heads, columns, reached = [1], [77], _below(trees[0], node)
    elif what == "decay":
        batch.dev_g[node, 1] = bad
        heads, reached = [1], _below(trees[0], node)
    else:
        batch.dev_b[node, 1] = bad
        heads, reached = [1], _below(trees[0], node)
    got = batch.tree().cpu()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    for i in reached:
        for h in heads:
            hit[i, h, columns] = True
    assert torch.equal(got[~hit], clean[~hit])
    if what == "decay" and bad == float("-inf"):
        assert torch.isfinite(got).all()
    else:
        assert not torch.isfinite(got[hit]).any()


def test_a_bad_state_stays_in_its_rows(device):
    batch = Batch(device, [ref.parents_of("any", 30, 14)], 2, 1, torch.float32, 61, rest=0)
    clean = batch.tree().cpu()
    batch.dev_pool[int(batch.slots[0]), 1, 40, 3] = float("nan")
    got = batch.tree().cpu()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[:, 1, 40] = True
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).any()


def test_bad_values_off_the_path_are_not_committed(device):
    tree = ref.parents_of("branches", 41)
    batch = Batch(device, [tree], 2, 1, torch.float32, 63)
    on_path = ref.path(tree, 40)
    for i in range(41):
        if i not in on_path:
            batch.mixed[i] = batch.g[i] = batch.b[i] = float("nan")
    for dev, cpu in ((batch.dev_mixed, batch.mixed), (batch.dev_g, batch.g),
                     (batch.dev_b, batch.b)):
        dev.copy_(cpu)
    batch.check_commit([40])


def test_states_past_four_gibibytes(device):
    """A slot and token rows whose byte offsets pass 2^32."""
    pool = torch.empty((4600, 16, 128, 128), device=device)  # 4.8 GB
    pool[4599] = 0.05
    mixed, g, b = tokens_of(3, 16, 16, 65)
    step = (1 << 24) - 8
    far = torch.empty((200 * step + 6144,), dtype=torch.bfloat16, device=device)
    rows = far.as_strided((200, 6144), (step, 1))
    rows[197:] = mixed.to(device)
    q, k, v = parts(mixed, 16, 16)
    dev = [rows[:, 2048 * i:2048 * (i + 1)].unflatten(1, (16, 128)) for i in range(3)]
    g_all, b_all = torch.zeros((200, 16)), torch.zeros((200, 16)).bfloat16()
    g_all[197:], b_all[197:] = g, b
    slots, parents = ints([-1, 4599], device), ints([-1] * 197 + [-1, 0, 0], device)
    tables = gdn.request_tables(ints([197, 3], device), slots, 200)
    rest = (g_all.to(device), b_all.to(device), parents)
    out = gdn.gated_delta_tree(*dev, *rest, tables, slots, pool)
    want, states = ref.tree(q, k, v, g, b, [-1, 0, 0], torch.full((16, 128, 128), 0.05))
    close(out[197:], want, BF16, "out")
    gdn.gated_delta_commit(*dev[1:], *rest, ints([0, 2], device), tables, slots, pool)
    close(pool[4599], states[2], FP32, "state")


def test_no_tokens(device):
    empty = [torch.empty((0, n, 128), dtype=torch.bfloat16, device=device) for n in (2, 2, 4)]
    rest = [torch.empty((0, 4), dtype=t, device=device) for t in (torch.float32, torch.bfloat16)]
    slots, pool = ints([0, 1], device), torch.ones((2, 4, 128, 128), device=device)
    tables = gdn.request_tables(ints([0, 0], device), slots, 0)
    out = gdn.gated_delta_tree(*empty, *rest, ints([], device), tables, slots, pool)
    assert out.shape == (0, 4, 128)
    gdn.gated_delta_commit(*empty[1:], *rest, ints([], device), ints([0, -1], device), tables,
                           slots, pool)
    assert (pool == 1).all()


def test_slices_that_start_at_any_element(device):
    """Parents, log decays and strengths may be slices of longer ones."""
    batch = Batch(device, [ref.parents_of("any", 21, 15)], 3, 1, torch.float32, 67, rest=0)
    whole = batch.tree()
    later = Batch(device, [ref.parents_of("any", 21, 15)], 3, 1, torch.float32, 67, rest=0)
    for name in ("dev_parents", "dev_g", "dev_b"):
        t = getattr(later, name)
        longer = torch.zeros((t.shape[0] + 1, *t.shape[1:]), dtype=t.dtype, device=device)
        longer[1:] = t
        setattr(later, name, longer[1:])
    assert torch.equal(later.tree(), whole)
    for b in (batch, later):
        b.commit([20])
    assert torch.equal(batch.dev_pool, later.dev_pool)


def test_side_stream_and_graph_replays(device):
    """Calls go to the current stream; a captured tree and commit replay, each from a pool
    and trees that were changed in between."""
    batch = Batch(device, [ref.parents_of("any", n, 16) for n in (20, 5, 64)], 4, 2,
                  torch.float32, 69, padded=False, rest=0)
    out = torch.zeros((89, 4, 128), dtype=torch.bfloat16, device=device)
    accepted = ints([19, 2, 63], device)

    def work():
        batch.tree(out)
        gdn.gated_delta_commit(*batch.inputs()[1:], batch.dev_parents, accepted, batch.tables,
                               batch.dev_slots, batch.dev_pool)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for take in range(3):
        batch.dev_pool.copy_(batch.pool + 0.01 * take)
        accepted.copy_(ints([19 - take, take - 1, 63 - 20 * take], device))
        start = batch.dev_pool.clone()
        work()
        torch.cuda.synchronize()
        eager = [out.clone(), batch.dev_pool.clone()]
        batch.dev_pool.copy_(start)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(batch.dev_pool, eager[1])


def test_results_do_not_vary_between_runs(device):
    batch = Batch(device, [ref.parents_of("any", n, 17) for n in (64, 33, 16, 5)], 8, 4,
                  torch.float32, 71, padded=False, rest=0)
    first = batch.tree()
    for _ in range(3):
        assert torch.equal(batch.tree(), first)


# ---------------------------------------------------------------- refusals

def test_refusals(device):
    batch = Batch(device, [ref.parents_of("chain", n) for n in (6, 4)], 4, 2, torch.float32, 73,
                  rest=0)
    q, k, v, g, b = batch.inputs()
    good = dict(queries=q, keys=k, values=v, log_decay=g, beta=b, parents=batch.dev_parents,
                tables=batch.tables, slot_ids=batch.dev_slots, pool=batch.dev_pool)
    gdn.gated_delta_tree(**good)
    t, d = good["tables"], device
    bad = [
        dict(queries=q.float()), dict(queries=q.cpu()), dict(queries=q[:9]),
        dict(keys=k[:, :1]), dict(values=v[:, :3]), dict(values=v.transpose(0, 1)),
        dict(log_decay=g.double()), dict(log_decay=g[:, :2]), dict(beta=b.float()),
        dict(parents=batch.dev_parents.long()), dict(parents=batch.dev_parents[:9]),
        dict(parents=batch.dev_parents.cpu()), dict(parents=batch.dev_parents.view(5, 2)),
        dict(tables=t._replace(offsets=t.offsets[:2])),
        dict(tables=t._replace(offsets=t.offsets.long())),
        dict(slot_ids=ints([0], d)), dict(slot_ids=batch.dev_slots.long()),
        dict(slot_ids=ints([], d)), dict(pool=batch.dev_pool.half()),
        dict(pool=batch.dev_pool[:, :2]), dict(pool=batch.dev_pool.transpose(2, 3)),
        dict(max_nodes=0), dict(max_nodes=65), dict(max_nodes=-1),
        dict(out=torch.zeros((10, 4, 128), device=d)),
        dict(out=torch.zeros((9, 4, 128), dtype=torch.bfloat16, device=d)),
        dict(values=v.clone().requires_grad_()), dict(pool=batch.dev_pool.clone().requires_grad_()),
    ]
    for change in bad:
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            gdn.gated_delta_tree(**{**good, **change})
    good.pop("queries")
    good["accepted"] = ints([5, 3], d)
    gdn.gated_delta_commit(**good)
    # (one key head for four values is an ordinary group without the queries' two)
    bad = [change for change in bad
           if not {"queries", "max_nodes", "out", "keys"} & set(change)]
    bad += [dict(keys=q[:, :0]), dict(keys=q.repeat(1, 2, 1)[:, :3].contiguous()), dict(accepted=ints([5], d)), dict(accepted=ints([5, 3], d).long()),
            dict(accepted=ints([5, 3], d).cpu())]
    for change in bad:
        with pytest.raises(RuntimeError, match="GDN State Codec"):
            gdn.gated_delta_commit(**{**good, **change})
