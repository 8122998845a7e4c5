"""The gated norm's fp32 outputs and gate gradients value by value, at gates of every
size.

With u = 2^-24, worst cases added up: 1 / sqrt of a 128-term mean 9 u, the gate's
sigmoid 8 u (exponential and reciprocal 2 u each, four operations), the output's four
products 4 u: 21 u, held to 24 u.  d_gate has four operations more and is held to 32 u,
away from -1.28, where the slope's two terms cancel."""

from __future__ import annotations

import pytest
import torch

import delta_reference as ref
import gdn_state_codec as gdn

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("low,high", [(-2.0, 2.0), (-20.0, -2.0), (-80.0, -20.0), (2.0, 80.0)])
def test_gated_norm_values(device, low, high):
    gen = torch.Generator().manual_seed(91)
    x, d = (torch.randn((64, 128), generator=gen) for _ in range(2))
    gate = low + (high - low) * torch.rand((64, 128), generator=gen)
    weight = 1.0 + 0.2 * torch.randn(128, generator=gen)
    leaves = [t.to(device).requires_grad_() for t in (x, gate, weight)]
    out = gdn.gated_norm(*leaves)
    d_gate = torch.autograd.grad([out], leaves, [d.to(device)])[1].double().cpu()
    want = ref.norm(x, weight, ref.silu(gate), 1e-6)
    off = ((out.detach().double().cpu() - want) / want).abs().max() / U
    want = ref.norm_gradients(x, weight, ref.silu(gate), d, 1e-6)[2] * ref.silu_slope(gate)
    slope_off = ((d_gate - want) / want).abs()[(gate + 1.28).abs() > 0.5].max() / U
    print(f"{low}..{high}: {float(off):.3g} u, {float(slope_off):.3g} u", flush=True)
    assert off <= 24 and slope_off <= 32


def test_gates_without_end(device):
    """A gate of +inf passes its value on times inf, -inf and NaN give NaN, and gates whose
    sigmoid underflows zero or less than the smallest normal number."""
    x, weight = torch.ones((1, 128), device=device), torch.ones(128, device=device)
    gate = torch.zeros((1, 128), device=device)
    ends = torch.tensor([float("inf"), 3.0e38, 200.0, -200.0, -3.0e38, float("-inf"),
                         float("nan")])
    gate[0, :7] = ends.to(device)
    out = gdn.gated_norm(x, gate, weight, eps=0.0).cpu()[0]
    assert torch.equal(out[:3], ends[:3])
    assert (out[3:5].abs() < 2.0 ** -126).all()
    assert torch.isnan(out[5:7]).all() and (out[7:] == 0).all()
