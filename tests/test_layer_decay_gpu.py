"""Log decays' gradients where decays are strong, against float64.

A log decay's gradient is the sum of what crosses its token: products of a gradient
after it and a write before it, each with the decay between them.  Each such product
is two dots of 128 fp32 terms on values that are good to 20 x 2^-24 (test_layer_gpu):
2^-17 of their sum's 2-norm.  For one token, <dS, S> is held to 2^-18 |dS| |S|, whose
terms it adds; both factors are as large as the decay leaves them."""

from __future__ import annotations

import pytest
import torch

import delta_reference as ref
import gdn_state_codec as gdn

pytestmark = pytest.mark.gpu

BATCHES = [([70, 0, 129], 4, 2), ([200, 1, 64, 0, 130, 63], 6, 3)]  # both forms of the scans


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def inputs(lengths, heads, key_heads, seed):
    gen = torch.Generator().manual_seed(seed)
    total = sum(lengths)
    q, k, v = (torch.randn((total, n, 128), generator=gen).bfloat16()
               for n in (key_heads, key_heads, heads))
    log_decay = -0.05 * torch.rand((total, heads), generator=gen)
    beta = torch.sigmoid(torch.randn((total, heads), generator=gen)).bfloat16()
    shape = (len(lengths), heads, 128, 128)
    initial = 0.1 * torch.randn(shape, generator=gen)
    d_out = torch.randn((total, heads, 128), generator=gen).bfloat16()
    return [q, k, v, log_decay, beta, initial], d_out, 0.1 * torch.randn(shape, generator=gen)


def gradients(device, x, lengths, d_out, d_final):
    leaves = [t.to(device).requires_grad_() for t in x]
    tables = gdn.request_tables(ints(lengths, device), ints(range(len(lengths)), device),
                                sum(lengths))
    outs = gdn.gated_delta_rule(*leaves[:5], tables, leaves[5])
    grads = torch.autograd.grad(outs, leaves, [d_out.to(device), d_final.to(device)])
    return [t.double().cpu() for t in grads]


def sizes(x, lengths, d_out, d_final, scale=128 ** -0.5):
    """|dS| |S| of each token and head: its state after its decay and the gradient there."""
    q, k, v, log_decay, beta, initial = x
    q, k = ref.expanded(q, k, v.shape[1] // q.shape[1], scale, True)
    v, a, b, d_out = v.double(), log_decay.double().exp(), beta.double(), d_out.double()
    size = torch.zeros_like(a)
    at = 0
    for n, length in enumerate(lengths):
        state, kept = initial[n].double(), []
        for t in range(at, at + length):
            state = state * a[t][:, None, None]
            kept.append(state)
            error = v[t] - torch.matmul(state, k[t][:, :, None])[..., 0]
            state = state + (b[t][:, None] * error)[:, :, None] * k[t][:, None, :]
        d = d_final[n].double()
        for t in range(at + length - 1, at - 1, -1):
            d = d + d_out[t][:, :, None] * q[t][:, None, :]
            d = d - (b[t][:, None] * torch.matmul(d, k[t][:, :, None])[..., 0])[:, :, None] * \
                k[t][:, None, :]
            size[t] = d.norm(dim=(1, 2)) * kept[t - at].norm(dim=(1, 2))
            d = d * a[t][:, None, None]
        at += length
    return size


@pytest.mark.parametrize("lengths,heads,key_heads", BATCHES)
@pytest.mark.parametrize("decay", [-1.0, -6.0, -12.0, -20.0])
def test_every_decay_strong(device, lengths, heads, key_heads, decay):
    x, d_out, d_final = inputs(lengths, heads, key_heads, 81)
    x[3].fill_(decay)
    got = gradients(device, x, lengths, d_out, d_final)[3]
    want = ref.rule_gradients(*x[:5], lengths, x[5], d_out, d_final)[3]
    off = float((got - want).norm() / want.norm())
    print(f"{decay}: {off:.3g}", flush=True)
    assert off <= 2.0 ** -17


@pytest.mark.parametrize("lengths,heads,key_heads", BATCHES)
def test_some_decays_strong(device, lengths, heads, key_heads):
    """Strong ones among weak ones, at a chunk's first and last token and inside."""
    x, d_out, d_final = inputs(lengths, heads, key_heads, 83)
    for i, t in enumerate((0, 13, 63, 64, 69, 100, 127, 198)):
        x[3][t] = -6.0 - 4.0 * (i % 4)
    got = gradients(device, x, lengths, d_out, d_final)[3]
    want = ref.rule_gradients(*x[:5], lengths, x[5], d_out, d_final)[3]
    off = (got - want).abs() / sizes(x, lengths, d_out, d_final)
    print(f"{float(off.max()):.3g}", flush=True)
    assert (off <= 2.0 ** -18).all()


@pytest.mark.parametrize("lengths,heads,key_heads", BATCHES)
def test_decays_of_minus_infinity(device, lengths, heads, key_heads):
    """Nothing passes such a token: its own gradient is zero, the others' as the formula's."""
    x, d_out, d_final = inputs(lengths, heads, key_heads, 85)
    gone = torch.tensor([0, 20, 63, 64, 140])
    x[3][gone] = float("-inf")
    x[3][100, 1] = -3.0e38
    got = gradients(device, x, lengths, d_out, d_final)
    want = ref.rule_gradients(*x[:5], lengths, x[5], d_out, d_final)
    assert (got[3][gone] == 0).all() and got[3][100, 1] == 0
    off = float((got[3] - want[3]).norm() / want[3].norm())
    assert off <= 2.0 ** -17
    for name, a, b, bound in zip(("q", "k", "v"), got, want, [2.0 ** -9 + 2.0 ** -12] * 3):
        b = b.bfloat16().double()
        assert float((a - b).norm()) <= bound * float(b.norm()), name
    b = want[4].bfloat16().double()
    assert float((got[4] - b).norm()) <= (2.0 ** -9 + 2.0 ** -12) * float(b.norm())
    assert float((got[5] - want[5]).norm()) <= 2.0 ** -18 * float(want[5].norm())
