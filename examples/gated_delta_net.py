"""A small gated-delta-net, trained and served with the layer operators.

Blocks of residual_norm -> projections -> the gated delta rule -> gated_norm ->
projection learn to repeat the token LAG positions back, on packed batches of
ragged sequences (request_tables, gated_delta_rule and the norms, with their
gradients).  The trained blocks are then served: a ragged batch of prompts fills
the state pool (gated_delta_prefill), the answers are decoded token by token
(gated_delta_step) and by trees of drafted tokens on a fork of the prompts' slots
(slot_moves, copy_slots, gated_delta_tree, gated_delta_commit), the pool goes
through the int8 codec and back (pool_encode, pool_decode) as a hibernated request's
would, and one request is decoded by GdnStateCodecRuntime's windowed int8 steps from
the same pool.

    python examples/gated_delta_net.py [--steps N]

Data are random; the short convolution that such layers often have before the rule
is left out.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

PACKAGE_ROOT = Path(__file__).resolve().parents[1] / "gdn-state-codec_amd"
if str(PACKAGE_ROOT) not in sys.path:
    sys.path.insert(0, str(PACKAGE_ROOT))

import gdn_state_codec as gdn  # noqa: E402

LAG = 3
DIM = 128


class Block(torch.nn.Module):
    """One layer: weights fp32, products and activations bf16."""

    def __init__(self, hidden: int, heads: int, key_heads: int) -> None:
        super().__init__()
        self.heads, self.key_heads = heads, key_heads
        self.widths = (key_heads * DIM, key_heads * DIM, heads * DIM)

        def weight(rows, columns):
            return torch.nn.Parameter(torch.randn(rows, columns) * columns ** -0.5)

        self.mixed = weight(sum(self.widths), hidden)      # queries, keys, values
        self.gate = weight(heads * DIM, hidden)
        self.rates = weight(2 * heads, hidden)             # decays and write strengths
        self.out = weight(hidden, heads * DIM)
        self.log_rate = torch.nn.Parameter(torch.linspace(-4.0, 0.0, heads))
        self.norm = torch.nn.Parameter(torch.ones(hidden))
        self.rule_norm = torch.nn.Parameter(torch.ones(DIM))

    def project(self, x: torch.Tensor):
        """The rule's inputs (queries, keys and values stay slices of one
        projection) and the gate."""
        tokens = x.shape[0]
        q, k, v = (part.view(tokens, -1, DIM) for part in
                   F.linear(x, self.mixed.bfloat16()).split(self.widths, dim=1))
        decay, strength = F.linear(x, self.rates.bfloat16()).float().split(self.heads, dim=1)
        log_decay = -torch.exp(self.log_rate) * F.softplus(decay)
        beta = torch.sigmoid(strength).bfloat16()
        gate = F.linear(x, self.gate.bfloat16()).view(tokens, self.heads, DIM)
        return (q, k, v, log_decay, beta), gate

    def forward(self, x, stream, rule):
        """(this block's output, the residual stream with the last block's output);
        ``rule`` maps the rule's inputs to its outputs [tokens,heads,128]."""
        x, stream = gdn.residual_norm(x, stream, self.norm)
        inputs, gate = self.project(x)
        x = gdn.gated_norm(rule(*inputs), gate, self.rule_norm)
        return F.linear(x.flatten(1), self.out.bfloat16()), stream


class Net(torch.nn.Module):
    def __init__(self, hidden: int = 256, layers: int = 2, heads: int = 4,
                 key_heads: int = 2) -> None:
        super().__init__()
        self.heads, self.key_heads = heads, key_heads
        self.blocks = torch.nn.ModuleList(Block(hidden, heads, key_heads)
                                          for _ in range(layers))
        self.norm = torch.nn.Parameter(torch.ones(hidden))

    def forward(self, tokens: torch.Tensor, rules) -> torch.Tensor:
        """bf16 [T,hidden] -> bf16 [T,hidden]; ``rules`` gives each layer's rule."""
        x, stream = tokens, torch.zeros(tokens.shape, device=tokens.device)
        for block, rule in zip(self.blocks, rules):
            x, stream = block(x, stream, rule)
        return gdn.residual_norm(x, stream, self.norm)[0]

    def train_rules(self, tables):
        return [lambda *inputs: gdn.gated_delta_rule(*inputs, tables)[0]] * len(self.blocks)

    def prefill_rules(self, tables, slots, fresh, pool):
        """Each layer's rule over whole prompts, its states left in ``pool``
        [layers,slots,heads,128 value,128 key]."""
        return [lambda *inputs, states=states:
                gdn.gated_delta_prefill(*inputs, tables, slots, states, resume=fresh)
                for states in pool]

    def tree_rules(self, parents, tables, slots, pool, seen: list):
        """Each layer's rule over trees of drafted tokens, from states that stay as they are;
        ``seen`` gets what committing an accepted path takes."""
        def rule(states):
            def outputs(*inputs):
                seen.append((states, inputs[1:]))
                return gdn.gated_delta_tree(*inputs, parents, tables, slots, states)
            return outputs
        return [rule(states) for states in pool]

    def step_rules(self, slots, pool):
        return [lambda *inputs, states=states: gdn.gated_delta_step(*inputs, states, slots)
                for states in pool]


def packed(lengths, hidden: int, device, generator):
    """Random tokens of a packed batch, what each should answer (the token LAG
    before it), which of them have an answer, and the batch's tables."""
    total = sum(lengths)
    tokens = torch.randn((total, hidden), generator=generator).bfloat16()
    place = torch.cat([torch.arange(n) for n in lengths])
    known = place >= LAG
    answers = torch.where(known[:, None], tokens.roll(LAG, 0).float(), 0.0)
    slots = torch.arange(len(lengths), dtype=torch.int32, device=device)
    tables = gdn.request_tables(torch.tensor(lengths, dtype=torch.int32, device=device),
                                slots, total)
    return tokens.to(device), answers.to(device), known.to(device), slots, tables


def train(net: Net, steps: int, device, generator, rate: float = 3e-3) -> list[float]:
    """The loss of each step: the mean squared error against the answers (of
    variance 1)."""
    optimizer = torch.optim.Adam(net.parameters(), lr=rate)
    losses = []
    for _ in range(steps):
        lengths = torch.randint(1, 200, (6,), generator=generator).tolist()
        tokens, answers, known, _, tables = packed(lengths, net.norm.numel(), device, generator)
        out = net(tokens, net.train_rules(tables)).float()
        loss = ((out - answers)[known] ** 2).sum() / (known.sum() * out.shape[1]).clamp(min=1)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def decode_by_trees(net: Net, rows, lengths, answers: int, slots, pool, generator):
    """The answers' outputs by trees of drafted tokens: each tree is a chain of the next
    two tokens (the last answer's, where their number is odd, of it alone), which are
    accepted, and a wrong guess beside each of them."""
    device, hidden = pool.device, rows[0].shape[1]

    def ints(x):
        return torch.tensor(x * len(rows), dtype=torch.int32, device=device)

    outs = []
    for i in range(0, answers, 2):
        depth = min(2, answers - i)
        nodes = 2 * depth
        wrong = torch.randn((len(rows), depth, hidden), generator=generator).bfloat16().to(device)
        tokens = torch.cat([torch.stack([row[n + i:n + i + depth], guess], 1).flatten(0, 1)
                            for row, n, guess in zip(rows, lengths, wrong)])
        parents, accepted = ints([-1, -1, 0, 0][:nodes]), ints([nodes - 2])
        tables = gdn.request_tables(ints([nodes]), slots, nodes * len(rows))
        seen = []
        out = net(tokens, net.tree_rules(parents, tables, slots, pool, seen))
        outs.append(out.view(len(rows), nodes, hidden)[:, ::2])
        for states, inputs in seen:
            gdn.gated_delta_commit(*inputs, parents, accepted, tables, slots, states)
    return torch.cat(outs, 1)  # [requests,answers,hidden]


def apart(x: torch.Tensor, y: torch.Tensor) -> float:
    x, y = x.double(), y.double()
    return float((x - y).norm() / y.norm())


@torch.no_grad()
def serve(net: Net, lengths, answers: int, device, generator) -> dict[str, float]:
    """Prompts of ``lengths`` and then ``answers`` tokens of each request: how far the
    served outputs are from those of one pass over everything."""
    hidden = net.norm.numel()
    requests = len(lengths)
    whole = [n + answers for n in lengths]
    tokens, _, _, _, tables = packed(whole, hidden, device, generator)
    expected = [part[n:] for part, n in
                zip(net(tokens, net.train_rules(tables)).split(whole), lengths)]
    rows = list(tokens.split(whole))

    # Slots of a pool with room for more requests, in no particular order.
    slots = (torch.arange(requests, dtype=torch.int32) * 3 + 2).flip(0).contiguous().to(device)
    pool = torch.randn((len(net.blocks), 3 * requests + 2, net.heads, DIM, DIM), device=device)
    fresh = torch.zeros(requests, dtype=torch.int32, device=device)
    prompts = torch.cat([row[:n] for row, n in zip(rows, lengths)])
    tables = gdn.request_tables(torch.tensor(lengths, dtype=torch.int32, device=device), slots,
                                prompts.shape[0])
    net(prompts, net.prefill_rules(tables, slots, fresh, pool))
    after_prompts = pool.clone()

    def decode(pool):
        outs = [net(torch.stack([row[n + i] for row, n in zip(rows, lengths)]),
                    net.step_rules(slots, pool)) for i in range(answers)]
        return torch.stack(outs, 1)  # [requests,answers,hidden]

    expected = torch.stack(expected)
    # The same by trees, on slots that the prompts' states were forked to.
    forked = pool.clone()
    ends = (slots + 1).contiguous()
    gdn.copy_slots(list(forked), gdn.slot_moves(slots, ends, pool.shape[1]))
    off = {"decoded": apart(decode(pool), expected),
           "decoded by trees": apart(decode_by_trees(net, rows, lengths, answers, ends, forked,
                                                     generator), expected)}

    codes = gdn.pool_encode(after_prompts, slots, gdn.LAYOUT_VALUE_KEY)
    restored = torch.zeros_like(after_prompts)
    gdn.pool_decode(*codes, slots, restored, gdn.LAYOUT_VALUE_KEY)
    off["decoded from int8 states"] = apart(decode(restored), expected)

    # One request by the windowed int8 steps, which take unit queries and keys.
    runtimes = [gdn.GdnStateCodecRuntime() for _ in net.blocks]
    slot = int(slots[0])

    def windowed(runtime, states):
        def rule(q, k, v, log_decay, beta):
            q, k = (F.normalize(t.float(), dim=-1).bfloat16() for t in (q, k))
            return runtime.step(states, slot, q[None], k[None], v[None].contiguous(),
                                log_decay[None], beta[None], DIM ** -0.5)[0]
        return rule

    rules = [windowed(*pair) for pair in zip(runtimes, after_prompts)]
    outs = [net(rows[0][lengths[0] + i][None], rules) for i in range(answers)]
    off["decoded by windowed int8 steps"] = apart(torch.cat(outs), expected[0])
    for runtime in runtimes:
        runtime.close()
    return off


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    steps = parser.parse_args().steps
    if not torch.cuda.is_available():
        raise SystemExit("this example needs a GPU")
    device = torch.device("cuda:0")
    generator = torch.Generator().manual_seed(7)
    torch.manual_seed(7)
    net = Net().to(device)
    losses = train(net, steps, device, generator)
    for i in range(0, steps, max(1, steps // 10)):
        print(f"step {i}: loss {losses[i]:.4f}", flush=True)
    for what, off in serve(net, [70, 1, 260, 33], 20, device, generator).items():
        print(f"{what}: {off:.2e} from one pass over everything", flush=True)


if __name__ == "__main__":
    main()
