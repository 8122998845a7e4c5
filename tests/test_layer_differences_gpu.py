"""Gradients against differences of the kernels' own values, for the inputs that
test_layer_gpu does not difference.

bf16 inputs move by what their rounding leaves of a step, which is known exactly; a
gradient g along a move of random values is |g| times its deviation.
* Outputs are linear in queries that are not normalized, and final states in values:
  any move will do, and what remains is the rounding of gradients and outputs to bf16
  (2^-9 each, independent): 2^-6.
* Keys and strengths: a step of h = 0.02 of a token's own size through the product of 64
  tokens' factors leaves (h sqrt(64))^2 / 6 = 0.4% in a central difference, and the middle
  of two rounded points is up to 2^-9 of a value off, through as many factors 64^0.5 2^-9 =
  1.6%: 3%.
* The residual norm in fp32: h = 1e-2 leaves 1e-4, and 2^-22 of the value over h."""

from __future__ import annotations

import pytest
import torch

import gdn_state_codec as gdn

pytestmark = pytest.mark.gpu

HEADS, KEY_HEADS = 4, 2


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.fixture
def batch(device):
    gen = torch.Generator().manual_seed(101)

    def made(*shape):
        return torch.randn(shape, generator=gen).to(device)

    lengths = [64, 40]
    total = sum(lengths)
    x = {"queries": made(total, KEY_HEADS, 128).bfloat16(),
         "keys": made(total, KEY_HEADS, 128).bfloat16(),
         "values": made(total, HEADS, 128).bfloat16(),
         "log_decay": -0.05 * made(total, HEADS).abs(),
         "beta": torch.sigmoid(made(total, HEADS)).bfloat16()}
    tables = gdn.request_tables(ints(lengths, device), ints([0, 1], device), total)
    start = 0.1 * made(2, HEADS, 128, 128)
    return x, tables, start, made


@pytest.mark.parametrize("name,output,normalize,bound", [
    ("queries", 0, False, 2.0 ** -6), ("values", 1, True, 2.0 ** -6), ("keys", 1, True, 0.03),
    ("beta", 1, True, 0.03)])
def test_rule_differences(batch, name, output, normalize, bound):
    x, tables, start, made = batch
    if not normalize:
        x["keys"] = x["keys"] * 0.08
    weight = made(*(x["values"].shape if output == 0 else start.shape))
    if output == 0:
        weight = weight.bfloat16()

    def value(moved):
        return gdn.gated_delta_rule(**{**x, name: moved}, tables=tables, initial=start,
                                    normalize=normalize)[output]

    leaf = x[name].clone().requires_grad_()
    grad, = torch.autograd.grad([value(leaf)], [leaf], [weight])
    way = made(*leaf.shape)
    with torch.no_grad():
        if bound < 0.02:  # linear
            points = [x[name], (x[name].float() + way).bfloat16()]
        else:
            points = [(x[name].float() * (1 + h * way)).bfloat16() for h in (-0.02, 0.02)]
        ends = [(value(p).double() * weight.double()).sum() for p in points]
    move = points[1].double() - points[0].double()
    got, want = float(ends[1] - ends[0]), float((grad.double() * move).sum())
    size = float((grad.double() * move).norm())
    print(f"{name}: {got} {want} {size}", flush=True)
    assert abs(got - want) <= bound * max(abs(want), size)


@pytest.mark.parametrize("width", [128, 1000, 4096])
@pytest.mark.parametrize("both", [False, True])
def test_residual_norm_differences(device, width, both):
    gen = torch.Generator().manual_seed(103)
    x, residual, d, d_sum = (torch.randn((5, width), generator=gen).to(device) for _ in range(4))
    weight = (1.0 + 0.2 * torch.randn(width, generator=gen)).to(device)
    ds = [d, d_sum if both else torch.zeros_like(d_sum)]
    inputs = [x, residual, weight]
    leaves = [t.clone().requires_grad_() for t in inputs]
    outs = gdn.residual_norm(*leaves, scale=0.75)
    grads = torch.autograd.grad(outs if both else outs[:1], leaves, ds if both else ds[:1])
    for i in range(3):
        way = torch.randn(leaves[i].shape, generator=gen).to(device)
        up, down = list(inputs), list(inputs)
        up[i], down[i] = up[i] + 1e-2 * way, down[i] - 1e-2 * way

        def value(a):
            return sum(float((o.double() * w).sum())
                       for o, w in zip(gdn.residual_norm(*a, scale=0.75), ds))

        slope = (value(up) - value(down)) / 2e-2
        want, size = float((grads[i].double() * way).sum()), float(grads[i].norm())
        print(f"{i}: {slope} {want} {size}", flush=True)
        assert abs(slope - want) <= 2e-3 * max(abs(want), size)
