"""What the rule's outputs are good to where their terms cancel, and how far a NaN or an
infinity goes."""

from __future__ import annotations

import pytest
import torch

import delta_reference as ref
import gdn_state_codec as gdn

pytestmark = pytest.mark.gpu

FORMS = [(2, 2, 1), (12, 4, 2)]  # requests, heads, key heads: both forms of the scans


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.mark.parametrize("requests,heads,key_heads", FORMS)
@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("size", [1.0, 30.0, 1000.0])
def test_outputs_whose_terms_cancel(device, requests, heads, key_heads, train, size):
    """Keys and queries all alike, whole writes (beta 1) over a start state `size` times the
    values: an output q S0 + sum_j P_ij E_j is a value, its terms are `size` times that.  The
    terms are good to 2^-15, the output is rounded to bf16 (2^-9)."""
    gen = torch.Generator().manual_seed(95)
    length = 60
    total = requests * length
    k = torch.randn((1, key_heads, 128), generator=gen).bfloat16().expand(total, -1, -1)
    v = torch.randn((total, heads, 128), generator=gen).bfloat16()
    log_decay, beta = torch.zeros(total, heads), torch.ones(total, heads).bfloat16()
    start = size * torch.randn((requests, heads, 128, 128), generator=gen)
    x = [t.contiguous().to(device) for t in (k, k, v, log_decay, beta)]
    slots = ints(range(requests), device)
    tables = gdn.request_tables(ints([length] * requests, device), slots, total)
    pool = start.to(device)
    out = (gdn.gated_delta_rule(*x, tables, pool, scale=1.0)[0] if train else
           gdn.gated_delta_prefill(*x, tables, slots, pool, scale=1.0))
    out = out.double().cpu()

    want, _ = ref.rule(k, k, v, log_decay, beta, [length] * requests, start, 1.0)
    unit = ref.unit(k[0].double())[0].repeat_interleave(heads // key_heads, 0)  # [heads,128]
    along = (unit * unit).sum(-1)[:, None]
    shape = (requests, length, heads, 128)
    terms = (start.double().abs() * unit.abs()[:, None]).sum(-1)[:, None].expand(shape).clone()
    state = torch.matmul(start.double(), unit[:, :, None])[..., 0]  # S k, [requests,heads,128]
    for t in range(length):
        error = v.view(shape)[:, t].double() - state
        state = state + along * error
        terms[:, t:] += (along * error).abs()[:, None]
    bound = 2.0 ** -15 * terms.reshape(out.shape) + 2.0 ** -8 * want.abs()
    print(f"{float(((out - want).abs() / bound).max()):.3g}", flush=True)
    assert ((out - want).abs() <= bound).all()


@pytest.mark.parametrize("requests,heads,key_heads", FORMS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("place", range(5))
def test_bad_values_stay_in_their_request(device, requests, heads, key_heads, bad, place):
    """A NaN or an infinity in one token reaches its own request from its 64-token chunk
    on; other requests, and the chunks before, keep every bit."""
    gen = torch.Generator().manual_seed(97)
    lengths = [200] * requests
    total = sum(lengths)
    x = [torch.randn((total, n, 128), generator=gen).bfloat16()
         for n in (key_heads, key_heads, heads)]
    x += [-0.1 * torch.rand((total, heads), generator=gen),
          torch.sigmoid(torch.randn((total, heads), generator=gen)).bfloat16()]
    slots = ints(range(requests), device)
    tables = gdn.request_tables(ints(lengths, device), slots, total)
    start = torch.randn((requests, heads, 128, 128), generator=gen).to(device)

    def run():
        pool = start.clone()
        inputs = [t.to(device) for t in x]
        out = gdn.gated_delta_prefill(*inputs, tables, slots, pool)
        trained, final = gdn.gated_delta_rule(*inputs, tables, start)
        return [t.cpu() for t in (out, pool, trained, final)]

    clean = run()
    x[place][200 + 130].view(-1)[5 if place < 3 else 0] = bad
    got = run()
    for a, b in zip(got, clean):
        if a.shape[0] == total:
            assert torch.equal(a[:200 + 128], b[:200 + 128])
            assert torch.equal(a[400:], b[400:])
        else:
            keep = [i for i in range(requests) if i != 1]
            assert torch.equal(a[keep], b[keep])
