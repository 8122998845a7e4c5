"""The gated delta rule and the layer's norms in float64 on the CPU, token by
token and straight from their definitions, with their gradients: what the kernels
of ``gdn_state_codec.layer`` are held to."""

from __future__ import annotations

import torch

DIM = 128
UNIT_EPS = 1e-6


def tables(lengths, slots, max_tokens, rows):
    """offsets, chunk_offsets, chunks and order as lists."""
    offsets, first, chunks = [0], [0], []
    for r, length in enumerate(lengths):
        begin, end = offsets[-1], min(offsets[-1] + max(length, 0), max_tokens)
        chunks += [[r, t, min(64, end - t), slots[r]] for t in range(begin, end, 64)]
        offsets.append(end)
        first.append(len(chunks))
    order = sorted(range(len(lengths)), key=lambda r: first[r] - first[r + 1])
    return offsets, first, chunks + [[-1, 0, 0, -1]] * (rows - len(chunks)), order


def unit(x):
    r = ((x * x).sum(-1, keepdim=True) + UNIT_EPS) ** -0.5
    return x * r, r


def unit_gradient(x, r, d):
    return r * d - x * r ** 3 * (x * d).sum(-1, keepdim=True)


def expanded(queries, keys, group, scale, normalize):
    """Scaled unit queries and unit keys of every value head, float64."""
    q, k = queries.double(), keys.double()
    if normalize:
        q, k = unit(q)[0], unit(k)[0]
    return (q * scale).repeat_interleave(group, 1), k.repeat_interleave(group, 1)


def rule(queries, keys, values, log_decay, beta, lengths, initial, scale=DIM ** -0.5,
         normalize=True):
    """out [T,H,128] and final [N,H,128 value,128 key] in float64; tokens of no
    request get zeros.  S <- exp(g) S; e = v - S k; S <- S + b e k^T; o = S q."""
    heads = values.shape[1]
    q, k = expanded(queries, keys, heads // queries.shape[1], scale, normalize)
    v, a, b = values.double(), log_decay.double().exp(), beta.double()
    out = torch.zeros(values.shape, dtype=torch.float64)
    final = initial.double().clone()
    at = 0
    for n, length in enumerate(lengths):
        state = final[n]
        for t in range(at, at + length):
            state = state * a[t][:, None, None]
            error = v[t] - torch.matmul(state, k[t][:, :, None])[..., 0]
            state = state + (b[t][:, None] * error)[:, :, None] * k[t][:, None, :]
            out[t] = torch.matmul(state, q[t][:, :, None])[..., 0]
        final[n] = state
        at += length
    return out, final


def rule_gradients(queries, keys, values, log_decay, beta, lengths, initial, d_out, d_final,
                   scale=DIM ** -0.5, normalize=True):
    """Gradients of rule() by hand: d_queries, d_keys, d_values, d_log_decay, d_beta,
    d_initial, from the states of every token."""
    heads, key_heads = values.shape[1], queries.shape[1]
    group = heads // key_heads
    q, k = expanded(queries, keys, group, scale, normalize)
    v, a, b = values.double(), log_decay.double().exp(), beta.double()
    d_out = d_out.double()
    d_q, d_k, d_v = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    d_g, d_b = torch.zeros_like(a), torch.zeros_like(b)
    d_initial = d_final.double().clone()
    at = 0
    for n, length in enumerate(lengths):
        state, kept = initial[n].double(), []
        for t in range(at, at + length):
            state = state * a[t][:, None, None]
            error = v[t] - torch.matmul(state, k[t][:, :, None])[..., 0]
            kept.append((state, error))
            state = state + (b[t][:, None] * error)[:, :, None] * k[t][:, None, :]
        d_state = d_initial[n]
        for t in range(at + length - 1, at - 1, -1):
            before, error = kept[t - at]
            after = before + (b[t][:, None] * error)[:, :, None] * k[t][:, None, :]
            d_q[t] = torch.matmul(after.transpose(1, 2), d_out[t][:, :, None])[..., 0]
            d_state = d_state + d_out[t][:, :, None] * q[t][:, None, :]
            m = torch.matmul(d_state, k[t][:, :, None])[..., 0]
            d_b[t] = (m * error).sum(-1)
            d_error = b[t][:, None] * m
            d_v[t] = d_error
            d_k[t] = torch.matmul(d_state.transpose(1, 2),
                                  (b[t][:, None] * error)[:, :, None])[..., 0]
            d_k[t] -= torch.matmul(before.transpose(1, 2), d_error[:, :, None])[..., 0]
            d_state = d_state - d_error[:, :, None] * k[t][:, None, :]
            d_g[t] = (d_state * before).sum((1, 2))
            d_state = d_state * a[t][:, None, None]
        d_initial[n] = d_state
        at += length
    tokens = queries.shape[0]
    d_q = d_q.reshape(tokens, key_heads, group, DIM).sum(2) * scale
    d_k = d_k.reshape(tokens, key_heads, group, DIM).sum(2)
    if normalize:
        x, r = queries.double(), unit(queries.double())[1]
        d_q = unit_gradient(x, r, d_q)
        x, r = keys.double(), unit(keys.double())[1]
        d_k = unit_gradient(x, r, d_k)
    return d_q, d_k, d_v, d_g, d_b, d_initial


def norm(total, weight, through, eps):
    total = total.double()
    r = ((total * total).mean(-1, keepdim=True) + eps) ** -0.5
    return total * r * weight.double() * through


def silu(gate):
    gate = gate.double()
    return gate / (1.0 + torch.exp(-gate))


def norm_gradients(total, weight, through, d_out, eps):
    """d_total, d_weight and d_through of norm()."""
    total, weight, d = total.double(), weight.double(), d_out.double()
    width = total.shape[-1]
    r = ((total * total).mean(-1, keepdim=True) + eps) ** -0.5
    n = total * r
    d_n = d * weight * through
    d_total = r * (d_n - n * (d_n * n).mean(-1, keepdim=True))
    terms = (d * n * through).reshape(-1, width)
    return d_total, terms, d * n * weight


def silu_slope(gate):
    gate = gate.double()
    s = 1.0 / (1.0 + torch.exp(-gate))
    return s * (1.0 + gate * (1.0 - s))
