"""torch-facing dense operators of a gated-delta-net layer
(include/gdn_state_codec_layer.h): the tables of a ragged batch, the gated delta
rule for one token, for prefill and for training, and the norms around it.

Each function checks shapes, dtypes, devices and strides on the host (raising
``RuntimeError``, as the codec's do), launches the gfx950 kernels on torch's
current stream and raises ``RuntimeError`` on a nonzero status.  Nothing here
waits for the GPU: lengths, slot ids and tables stay on the device.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from ._native import RuleStruct, native

DIM = 128
CHUNK = 64             # tokens of a row of RequestTables.chunks
MAX_REQUESTS = 4096
QUERY_SCALE = DIM ** -0.5
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


# The current stream's handle, without the Stream object around it: a decode step
# is a few microseconds of host work, and this is asked for on every call.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _stream() -> int:
    return _raw_stream(_current_device())


def _fail(message: str) -> None:
    raise RuntimeError(f"GDN State Codec {message}")


def _launched(status: int, what: str) -> None:
    if status != 0:
        raise RuntimeError(f"GDN State Codec {what} launch failed: {status}")


# Messages are put together only when a check fails: formatting a tensor's shape
# and strides costs more than the whole call.

def _on_device(t: torch.Tensor, name: str) -> None:
    if t.get_device() != _current_device():
        _fail(f"{name} must be on the current GPU")


def _dense(t: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype) -> None:
    """A contiguous tensor of exactly this shape and type, on the current GPU."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        _fail(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}, got "
              f"{t.dtype} {tuple(t.shape)} with strides {tuple(t.stride())}")
    if t.get_device() != _current_device():
        _fail(f"{name} must be on the current GPU")


def _once() -> None:
    """In a backward pass: there is no gradient of the gradients."""
    if torch.is_grad_enabled():
        _fail("layer operators cannot be differentiated twice")


def _no_tangents(*tensors: torch.Tensor) -> None:
    """Refuses dual tensors, whose tangents a launch would drop."""
    if forward_ad._current_level >= 0 and any(
            forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        _fail("layer operators have no forward-mode derivative")


def _not_differentiated(what: str, *tensors: torch.Tensor) -> None:
    """Refuses tensors that ask for a gradient, which a call in place cannot give."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        _fail(f"{what} has no gradient: call it under torch.no_grad(), or "
              "gated_delta_rule to train")
    _no_tangents(*tensors)


class RequestTables(NamedTuple):
    """The device tables of a ragged batch of N requests (all int32)."""

    offsets: torch.Tensor        # [N+1] first token of each request, then their total
    chunk_offsets: torch.Tensor  # [N+1] first row of each request in `chunks`
    chunks: torch.Tensor         # [rows,4] request, first token, tokens, slot
    order: torch.Tensor          # [N] requests by falling chunk count


def table_rows(max_tokens: int, requests: int) -> int:
    """Rows of ``RequestTables.chunks``: what any lengths need at most."""
    return max_tokens // CHUNK + requests


def request_tables(lengths: torch.Tensor, slot_ids: torch.Tensor,
                   max_tokens: int) -> RequestTables:
    """The tables of a batch whose requests' tokens are packed in one
    ``max_tokens``-row buffer, from device int32 ``lengths`` and ``slot_ids`` [N]
    (N in 1..4096; slot -1: padding).  A negative length counts as 0, and tokens
    past ``max_tokens`` are cut off."""
    n = lengths.numel()
    if lengths.dim() != 1 or not 1 <= n <= MAX_REQUESTS:
        _fail(f"request lengths must be [1..{MAX_REQUESTS}]")
    _dense(lengths, "request lengths", (n,), torch.int32)
    _dense(slot_ids, "request slot ids", (n,), torch.int32)
    if not 0 <= max_tokens < 2 ** 31:
        _fail("request tables' max_tokens must be in 0..2^31-1")
    rows = table_rows(max_tokens, n)
    # One allocation; each table starts on a 16-byte boundary.
    buffer = torch.empty(4 * rows + 2 * (n // 4 * 4 + 4) + n, dtype=torch.int32,
                         device=lengths.device)
    chunks, offsets, _, chunk_offsets, _, order = buffer.split_with_sizes(
        (4 * rows, n + 1, 3 - n % 4, n + 1, 3 - n % 4, n))
    tables = RequestTables(offsets, chunk_offsets, chunks.view(rows, 4), order)
    _launched(native().request_tables_launch_v1(
        _stream(), lengths.data_ptr(), slot_ids.data_ptr(), n, max_tokens, rows,
        tables.offsets.data_ptr(), tables.chunk_offsets.data_ptr(), tables.chunks.data_ptr(),
        tables.order.data_ptr()), "request tables")
    return tables


# ------------------------------------------------------- the gated delta rule

def _token_rows(t: torch.Tensor, name: str, tokens: int) -> int:
    """Checks bf16 [tokens,heads,128] whose heads are packed; the distance between
    tokens may be any multiple of 8 elements (a slice of a fused projection).
    Returns that distance."""
    shape, (step, head_step, one) = t.shape, t.stride() if t.dim() == 3 else (0, 0, 0)
    if t.dtype is not torch.bfloat16 or len(shape) != 3 or shape[0] != tokens or \
            shape[1] < 1 or shape[2] != DIM:
        _fail(f"{name} must be bf16 [{tokens},heads,128], got {t.dtype} {tuple(shape)}")
    _on_device(t, name)
    width = shape[1] * DIM
    stride = step if tokens > 1 else width
    if one != 1 or (head_step != DIM and shape[1] != 1) or stride % 8 or stride < width:
        _fail(f"{name} must hold whole [heads,128] rows a multiple of 8 elements apart, got "
              f"strides {tuple(t.stride())}")
    return stride


def _rule_inputs(queries, keys, values, log_decay, beta):
    """Checks one batch of tokens; returns (tokens, value heads, key heads, strides)."""
    tokens = queries.shape[0] if queries.dim() else 0
    strides = (_token_rows(queries, "queries", tokens), _token_rows(keys, "keys", tokens),
               _token_rows(values, "values", tokens))
    heads, key_heads = values.shape[1], keys.shape[1]
    if queries.shape[1] != key_heads or heads % key_heads:
        _fail("queries and keys must have as many heads, and values a multiple of them")
    _dense(log_decay, "log decay", (tokens, heads), torch.float32)
    _dense(beta, "beta", (tokens, heads), torch.bfloat16)
    return tokens, heads, key_heads, strides


def _pool(pool: torch.Tensor, heads: int) -> int:
    if pool.dtype not in _TYPES or pool.dim() != 4 or pool.shape[0] < 1 or \
            pool.shape[1:] != (heads, DIM, DIM) or not pool.is_contiguous():
        _fail(f"state pool must be contiguous fp32 or bf16 [slots,{heads},128 value,128 key], "
              f"got {pool.dtype} {tuple(pool.shape)}")
    _on_device(pool, "state pool")
    return _TYPES[pool.dtype]


def gated_delta_step(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                     log_decay: torch.Tensor, beta: torch.Tensor, pool: torch.Tensor,
                     slot_ids: torch.Tensor, scale: float = QUERY_SCALE,
                     normalize: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """One token of the gated delta rule for each of B requests, on the dense
    states ``pool`` [slots,H,128 value,128 key] (fp32 or bf16, one layer), updated
    in place at ``slot_ids`` int32 [B] (distinct; outside the pool, as -1: padding,
    skipped, its output row left as it was).

    queries, keys bf16 [B,Hk,128], values bf16 [B,H,128] (rows of a fused
    projection are fine), log_decay fp32 and beta bf16 [B,H]; returns bf16
    [B,H,128].  ``normalize`` divides queries and keys by their 2-norm.  Not
    differentiable: inputs that require gradients are refused outside
    ``torch.no_grad()``."""
    batch, heads, key_heads, strides = _rule_inputs(queries, keys, values, log_decay, beta)
    pool_dtype = _pool(pool, heads)
    _not_differentiated("gated delta step", queries, keys, values, log_decay, beta, pool)
    _dense(slot_ids, "slot ids", (batch,), torch.int32)
    if out is None:
        out = torch.zeros((batch, heads, DIM), dtype=torch.bfloat16, device=values.device)
    else:
        _dense(out, "output", (batch, heads, DIM), torch.bfloat16)
    if batch:
        _launched(native().gated_delta_step_launch_v1(
            _stream(), queries.data_ptr(), keys.data_ptr(), values.data_ptr(),
            log_decay.data_ptr(), beta.data_ptr(), pool.data_ptr(), slot_ids.data_ptr(),
            out.data_ptr(), batch, pool.shape[0], heads, key_heads, *strides, pool_dtype,
            scale, normalize), "gated delta step")
    return out


def _check_tables(tables: RequestTables, tokens: int) -> int:
    """Checks that the tables are a batch's of `tokens` token rows; returns N."""
    requests = tables.order.numel()
    if not 1 <= requests <= MAX_REQUESTS:
        _fail(f"tables must hold 1..{MAX_REQUESTS} requests")
    for t, name, shape in ((tables.offsets, "offsets", (requests + 1,)),
                           (tables.chunk_offsets, "chunk_offsets", (requests + 1,)),
                           (tables.chunks, "chunks", (table_rows(tokens, requests), 4)),
                           (tables.order, "order", (requests,))):
        _dense(t, f"tables.{name}", shape, torch.int32)
    return requests


def workspace_bytes(tokens: int, requests: int, heads: int, key_heads: int,
                    train: bool = False) -> int:
    """Bytes of scratch that a prefill (or a forward and backward pass) takes."""
    return native().gated_delta_workspace_v1(table_rows(tokens, requests), heads, key_heads,
                                             train)


def _rule(queries, keys, values, log_decay, beta, tables, scale, normalize, workspace, train):
    """The checked argument struct of a whole-sequence call and its workspace."""
    tokens, heads, key_heads, strides = _rule_inputs(queries, keys, values, log_decay, beta)
    requests = _check_tables(tables, tokens)
    needed = workspace_bytes(tokens, requests, heads, key_heads, train)
    if workspace is None:
        workspace = torch.empty(needed, dtype=torch.uint8, device=values.device)
    else:
        if workspace.dtype is not torch.uint8 or not workspace.is_contiguous() or \
                workspace.numel() < needed:
            _fail(f"workspace must be contiguous uint8 of at least {needed} bytes")
        _on_device(workspace, "workspace")
    rule = RuleStruct(queries.data_ptr(), keys.data_ptr(), values.data_ptr(),
                      log_decay.data_ptr(), beta.data_ptr(), *strides,
                      tables.offsets.data_ptr(), tables.chunk_offsets.data_ptr(),
                      tables.chunks.data_ptr(), tables.order.data_ptr(), workspace.data_ptr(),
                      workspace.numel(), requests, tables.chunks.shape[0], tokens, heads,
                      key_heads, scale, normalize)
    return rule, workspace


def gated_delta_prefill(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                        log_decay: torch.Tensor, beta: torch.Tensor, tables: RequestTables,
                        slot_ids: torch.Tensor, pool: torch.Tensor,
                        resume: torch.Tensor | None = None, scale: float = QUERY_SCALE,
                        normalize: bool = True, workspace: torch.Tensor | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """The gated delta rule over the packed sequences of N requests, on the dense
    states ``pool`` [slots,H,128 value,128 key] (fp32 or bf16, one layer): request
    r starts from the state at ``slot_ids[r]`` (int32 [N], distinct; outside the
    pool, as -1: padding, skipped) where ``resume`` (int32 [N]) is nonzero or not
    given, from zeros where it is 0, and leaves its final state there.

    queries, keys bf16 [T,Hk,128], values bf16 [T,H,128] (rows of a fused
    projection are fine), log_decay fp32 and beta bf16 [T,H]; ``tables`` are
    :func:`request_tables`' for ``max_tokens`` T and the same slot ids.  Returns
    bf16 [T,H,128]; rows of no request, and padding's, stay as they were.
    ``workspace`` (uint8, :func:`workspace_bytes`) may be kept between calls; without
    ``out`` a call also clears a new one.  An output's terms are good to 2^-15 each (the
    states to fp32).  Not
    differentiable, as :func:`gated_delta_step`; :func:`gated_delta_rule` is."""
    rule, workspace = _rule(queries, keys, values, log_decay, beta, tables, scale, normalize,
                            workspace, False)
    heads = values.shape[1]
    pool_dtype = _pool(pool, heads)
    _not_differentiated("gated delta prefill", queries, keys, values, log_decay, beta, pool)
    _dense(slot_ids, "slot ids", (rule.requests,), torch.int32)
    if resume is not None:
        _dense(resume, "resume", (rule.requests,), torch.int32)
    if out is None:
        out = torch.zeros((rule.tokens, heads, DIM), dtype=torch.bfloat16, device=values.device)
    else:
        _dense(out, "output", (rule.tokens, heads, DIM), torch.bfloat16)
    _launched(native().gated_delta_prefill_launch_v1(
        _stream(), ctypes.byref(rule), slot_ids.data_ptr(),
        0 if resume is None else resume.data_ptr(), pool.data_ptr(), pool.shape[0], pool_dtype,
        out.data_ptr()), "gated delta prefill")
    return out


def _sizes(rule: RuleStruct) -> tuple:
    return rule.tokens, rule.requests, rule.value_heads, rule.key_heads


class _GatedDeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, queries, keys, values, log_decay, beta, initial, tables, scale, normalize):
        rule, workspace = _rule(queries, keys, values, log_decay, beta, tables, scale, normalize,
                                None, True)
        heads = rule.value_heads
        if initial is not None:
            _dense(initial, "initial states", (rule.requests, heads, DIM, DIM), torch.float32)
        out = torch.empty((rule.tokens, heads, DIM), dtype=torch.bfloat16, device=values.device)
        final = torch.empty((rule.requests, heads, DIM, DIM), dtype=torch.float32,
                            device=values.device)
        _launched(native().gated_delta_forward_launch_v1(
            _stream(), ctypes.byref(rule), 0 if initial is None else initial.data_ptr(),
            final.data_ptr(), out.data_ptr()), "gated delta forward")
        ctx.save_for_backward(queries, keys, values, log_decay, beta, *tables, workspace)
        ctx.sizes, ctx.scale, ctx.normalize = _sizes(rule), scale, normalize
        ctx.resumed = initial is not None
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    def backward(ctx, d_out, d_final):
        _once()
        # Under hooks on saved tensors (checkpointing, offloading) these are others than the
        # forward pass's, which may be gone: their addresses, strides and checks are taken anew.
        queries, keys, values, log_decay, beta, *tables, workspace = ctx.saved_tensors
        rule, _ = _rule(queries, keys, values, log_decay, beta, RequestTables(*tables), ctx.scale,
                        ctx.normalize, workspace, True)
        if _sizes(rule) != ctx.sizes:
            _fail("gated delta rule's saved tensors changed their shapes")
        shape = (rule.requests, rule.value_heads, DIM, DIM)
        if d_out is None:
            d_out = torch.zeros(values.shape, dtype=torch.bfloat16, device=values.device)
        d_out = _given(d_out, torch.bfloat16)
        if d_final is not None:
            d_final = _given(d_final, torch.float32)
        grads = [t.new_empty(t.shape) for t in (queries, keys, values, log_decay, beta)]
        d_initial = (torch.empty(shape, dtype=torch.float32, device=values.device)
                     if ctx.resumed else None)
        _launched(native().gated_delta_backward_launch_v1(
            _stream(), ctypes.byref(rule), d_out.data_ptr(),
            0 if d_final is None else d_final.data_ptr(), *(t.data_ptr() for t in grads),
            0 if d_initial is None else d_initial.data_ptr()), "gated delta backward")
        return *grads, d_initial, None, None, None


def gated_delta_rule(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                     log_decay: torch.Tensor, beta: torch.Tensor, tables: RequestTables,
                     initial: torch.Tensor | None = None, scale: float = QUERY_SCALE,
                     normalize: bool = True):
    """``(out, final)`` of the gated delta rule over the packed sequences of N
    requests, differentiable in every tensor: the inputs of
    :func:`gated_delta_prefill` with ``initial`` fp32 [N,H,128 value,128 key] (or
    None: zeros) in the pool's place.  out is bf16 [T,H,128] (zeros in rows of no
    request), final fp32 like initial.  The graph keeps a workspace of
    ``workspace_bytes(T, N, H, Hk, train=True)`` until its backward pass; under hooks on
    saved tensors (checkpointing, offloading) that and the inputs are the hooks'."""
    return _GatedDeltaRule.apply(queries, keys, values, log_decay, beta, initial, tables, scale,
                                 normalize)


# ------------------------------------------------------------------ the norms

def _rows_of(t: torch.Tensor, name: str, width: int) -> int:
    if t.dtype not in _TYPES or t.shape[-1] != width or not t.is_contiguous():
        _fail(f"{name} must be contiguous fp32 or bf16 [...,{width}], got {t.dtype} "
              f"{tuple(t.shape)}")
    _on_device(t, name)
    return t.numel() // width


def _given(d: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """An output's gradient as the kernels read it: dense, of its type, and on a 16-byte
    boundary (autograd hands over slices of larger gradients as they lie)."""
    if d.dtype is not dtype or not d.is_contiguous():
        d = d.to(dtype).contiguous()
    return d if d.data_ptr() % 16 == 0 else d.clone()


def _weight_sums(weight: torch.Tensor, rows: int):
    """The weight's gradient and the scratch its sum goes through."""
    parts = native().norm_partials_v1(rows, weight.numel())
    return torch.empty_like(weight), weight.new_empty(parts * weight.numel())


def _gated_norm(x, gate, weight, eps: float) -> torch.Tensor:
    out = torch.empty_like(x)
    if x.numel():
        _launched(native().gated_norm_launch_v1(
            _stream(), x.data_ptr(), gate.data_ptr(), weight.data_ptr(), out.data_ptr(),
            x.numel() // DIM, _TYPES[x.dtype], eps), "gated norm")
    return out


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, weight, eps):
        ctx.save_for_backward(x, gate, weight)
        ctx.eps = eps
        return _gated_norm(x, gate, weight, eps)

    @staticmethod
    def backward(ctx, d_out):
        _once()
        x, gate, weight = ctx.saved_tensors
        rows = x.numel() // DIM
        d_x, d_gate = torch.empty_like(x), torch.empty_like(x)
        if not rows:
            return d_x, d_gate, torch.zeros_like(weight), None
        d_out = _given(d_out, x.dtype)
        d_weight, partials = _weight_sums(weight, rows)
        _launched(native().gated_norm_backward_launch_v1(
            _stream(), x.data_ptr(), gate.data_ptr(), weight.data_ptr(), d_out.data_ptr(),
            d_x.data_ptr(), d_gate.data_ptr(), d_weight.data_ptr(), partials.data_ptr(), rows,
            _TYPES[x.dtype], ctx.eps), "gated norm backward")
        return d_x, d_gate, d_weight, None


def gated_norm(x: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor,
               eps: float = 1e-6) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight * gate * sigmoid(gate)`` over the last
    dimension (128): the norm after the rule, fused with the block's gate.

    x and gate [...,128] of one type (bf16 or fp32), weight fp32 [128]; the result
    has x's type.  Differentiable in all three."""
    if x.dim() < 1:
        _fail("gated norm input must have a last dimension of 128")
    _rows_of(x, "gated norm input", DIM)
    if gate.shape != x.shape or gate.dtype is not x.dtype:
        _fail("gate must have the input's shape and type")
    _rows_of(gate, "gate", DIM)
    _dense(weight, "gated norm weight", (DIM,), torch.float32)
    _no_tangents(x, gate, weight)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad
                                    or weight.requires_grad):
        return _GatedNorm.apply(x, gate, weight, eps)
    return _gated_norm(x, gate, weight, eps)


def _residual_norm(x, residual, weight, scale: float, eps: float):
    out, total = torch.empty_like(x), torch.empty_like(residual)
    if x.numel():
        width = x.shape[-1]
        _launched(native().residual_norm_launch_v1(
            _stream(), x.data_ptr(), residual.data_ptr(), weight.data_ptr(), out.data_ptr(),
            total.data_ptr(), x.numel() // width, width, _TYPES[x.dtype],
            _TYPES[residual.dtype], scale, eps), "residual norm")
    return out, total


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, scale, eps):
        out, total = _residual_norm(x, residual, weight, scale, eps)
        ctx.save_for_backward(total, weight)
        ctx.dtype, ctx.scale, ctx.eps = x.dtype, scale, eps
        ctx.set_materialize_grads(False)
        return out, total

    @staticmethod
    def backward(ctx, d_out, d_total):
        _once()
        total, weight = ctx.saved_tensors
        width = weight.numel()
        rows = total.numel() // width
        d_x, d_residual = torch.empty_like(total, dtype=ctx.dtype), torch.empty_like(total)
        if not rows:
            return d_x, d_residual, torch.zeros_like(weight), None, None
        d_out = torch.zeros_like(d_x) if d_out is None else _given(d_out, ctx.dtype)
        if d_total is not None:
            d_total = _given(d_total, total.dtype)
        d_weight, partials = _weight_sums(weight, rows)
        _launched(native().residual_norm_backward_launch_v1(
            _stream(), total.data_ptr(), weight.data_ptr(), d_out.data_ptr(),
            0 if d_total is None else d_total.data_ptr(), d_x.data_ptr(), d_residual.data_ptr(),
            d_weight.data_ptr(), partials.data_ptr(), rows, width, _TYPES[ctx.dtype],
            _TYPES[total.dtype], ctx.scale, ctx.eps), "residual norm backward")
        return d_x, d_residual, d_weight, None, None


def residual_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                  scale: float = 1.0, eps: float = 1e-6):
    """``(out, sum)`` with ``sum = residual + scale * x`` in the residual stream's
    type and ``out = sum / sqrt(mean(sum^2) + eps) * weight`` in x's: the norm
    before a block, fused with the scaled residual sum of the block before.

    x [...,D] and residual [...,D] bf16 or fp32 (each its own), weight fp32 [D], D
    a multiple of 8 up to 16384.  The norm is of the stored (rounded) sum.
    Differentiable in x, residual and weight."""
    if x.dim() < 1:
        _fail("residual norm input must have a last dimension")
    width = x.shape[-1]
    if width % 8 or not 0 < width <= 16384:
        _fail("residual norm width must be a multiple of 8 up to 16384")
    _rows_of(x, "residual norm input", width)
    if residual.shape != x.shape:
        _fail("the residual stream must have the input's shape")
    _rows_of(residual, "residual stream", width)
    _dense(weight, "residual norm weight", (width,), torch.float32)
    _no_tangents(x, residual, weight)
    if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad
                                    or weight.requires_grad):
        return _ResidualNorm.apply(x, residual, weight, scale, eps)
    return _residual_norm(x, residual, weight, scale, eps)
