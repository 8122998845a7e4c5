"""Batches without a token: torch gives an empty tensor no address, and each request is
still there with its state."""

from __future__ import annotations

import pytest
import torch

import gdn_state_codec as gdn
from gdn_state_codec import layer

pytestmark = pytest.mark.gpu


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def no_tokens(device, heads, key_heads):
    return [torch.empty((0, n, 128), dtype=torch.bfloat16, device=device)
            for n in (key_heads, key_heads, heads)] + [
        torch.empty((0, heads), dtype=t, device=device) for t in (torch.float32, torch.bfloat16)]


@pytest.mark.parametrize("requests,heads", [(4, 2), (12, 6)])  # both forms of the scans
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("given", [False, True])
def test_prefill_of_no_tokens(device, requests, heads, dtype, given):
    x = no_tokens(device, heads, heads // 2)
    pool = torch.randn((requests + 1, heads, 128, 128), device=device).to(dtype)
    slots = ints([requests - i for i in range(requests)], device)
    slots[1] = -1
    resume = ints([i % 2 for i in range(requests)], device)
    tables = gdn.request_tables(ints([0] * requests, device), slots, 0)
    more = dict(out=torch.empty_like(x[2]),
                workspace=torch.empty(layer.workspace_bytes(0, requests, heads, heads // 2),
                                      dtype=torch.uint8, device=device)) if given else {}
    want = pool.clone()
    for slot, go_on in zip(slots.tolist(), resume.tolist()):
        if slot >= 0 and not go_on:
            want[slot] = 0
    out = gdn.gated_delta_prefill(*x, tables, slots, pool, resume=resume, **more)
    assert out.shape == (0, heads, 128) and torch.equal(pool, want)
    gdn.gated_delta_prefill(*x, tables, slots, pool)  # all resume
    assert torch.equal(pool, want)


@pytest.mark.parametrize("requests,heads", [(4, 2), (12, 6)])
@pytest.mark.parametrize("resumed", [False, True])
def test_train_of_no_tokens(device, requests, heads, resumed):
    x = [t.requires_grad_() for t in no_tokens(device, heads, heads // 2)]
    shape = (requests, heads, 128, 128)
    initial = torch.randn(shape, device=device).requires_grad_() if resumed else None
    tables = gdn.request_tables(ints([0] * requests, device), ints(range(requests), device), 0)
    out, final = gdn.gated_delta_rule(*x, tables, initial)
    assert out.shape == (0, heads, 128)
    assert torch.equal(final, initial) if resumed else bool((final == 0).all())
    d_final = torch.randn(shape, device=device)
    wanted = x + ([initial] if resumed else [])
    grads = torch.autograd.grad([out, final], wanted, [torch.empty_like(out), d_final])
    for got, leaf in zip(grads, x):
        assert got.shape == leaf.shape
    if resumed:
        assert torch.equal(grads[5], d_final)
