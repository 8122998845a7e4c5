"""The float64 reference of the gated delta rule and of the norms: its gradients
against central differences of its values (float64, step 1e-5: the differences
are good to about 1e-9 of the largest term)."""

from __future__ import annotations

import pytest
import torch

import delta_reference as ref


def _inputs(lengths, heads, key_heads, seed):
    gen = torch.Generator().manual_seed(seed)
    total = sum(lengths)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    return (r(total, key_heads, 128), r(total, key_heads, 128), r(total, heads, 128),
            -torch.rand(total, heads, generator=gen, dtype=torch.float64),
            torch.rand(total, heads, generator=gen, dtype=torch.float64),
            0.1 * r(len(lengths), heads, 128, 128)), (r(total, heads, 128),
                                                      r(len(lengths), heads, 128, 128))


@pytest.mark.parametrize("normalize", [True, False])
def test_rule_gradients_are_the_differences(normalize):
    lengths, scale = [3, 0, 2], 0.3
    x, (d_out, d_final) = _inputs(lengths, 2, 1, 5)
    if not normalize:
        x = (x[0] * 0.1, x[1] * 0.1) + x[2:]

    def value(q, k, v, g, b, s):
        out, final = ref.rule(q, k, v, g, b, lengths, s, scale, normalize)
        return float((out * d_out).sum() + (final * d_final).sum())

    grads = ref.rule_gradients(*x[:5], lengths, x[5], d_out, d_final, scale, normalize)
    gen = torch.Generator().manual_seed(6)
    for i, grad in enumerate(grads):
        for _ in range(3):
            way = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
            up, down = list(x), list(x)
            up[i], down[i] = x[i] + 1e-5 * way, x[i] - 1e-5 * way
            slope = (value(*up) - value(*down)) / 2e-5
            want = float((grad * way).sum())
            assert abs(slope - want) <= 1e-6 * max(1.0, abs(want)), (i, slope, want)


def test_norm_gradients_are_the_differences():
    gen = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    x, w, z, d = r(4, 24), r(24), r(4, 24), r(4, 24)
    d_x, terms, d_through = ref.norm_gradients(x, w, ref.silu(z), d, 1e-3)
    grads = (d_x, terms.sum(0), d_through * ref.silu_slope(z))
    for i, grad in enumerate(grads):
        way = r(*grad.shape)
        up, down = [x, w, z], [x, w, z]
        up[i], down[i] = up[i] + 1e-5 * way, down[i] - 1e-5 * way
        value = lambda x, w, z: float((ref.norm(x, w, ref.silu(z), 1e-3) * d).sum())  # noqa: E731
        slope = (value(*up) - value(*down)) / 2e-5
        assert abs(slope - float((grad * way).sum())) <= 1e-7 * max(1.0, abs(slope))
