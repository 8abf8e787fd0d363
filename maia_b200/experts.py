"""Mixture-of-experts routing around gemm_grouped, and decode products with 4-bit weights.

    r = moe_route(logits, k)                        # experts and weights of every token, counts, balance loss
    plan = moe_plan(r.ids, experts)                 # rows of the m-grouped layout
    a = moe_dispatch(x, plan)
    y = gemm_grouped(a, w, plan.m_block_group)      # one matrix per expert
    out = moe_combine(y, r.weights, rows=plan.rows)

For a few tokens, without a layout: y = gemv_int4(x, q, scales, ids=r.ids); out = moe_combine(y, r.weights).
Every call is queued on the tensors' current CUDA stream (or `stream`) and allocates only its outputs,
through torch. No counterpart in the reference (kernel_lib has no GEMM and no routing).
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import (Int4Desc, KL_BF16, KL_F16, KL_F32, MoeRouteDesc, check, lib)

_FLOATS = {torch.bfloat16: KL_BF16, torch.float16: KL_F16, torch.float32: KL_F32}


class MoeRoute(NamedTuple):
    ids: torch.Tensor      # int32 [tokens, k], -1 = no expert
    weights: torch.Tensor  # fp32 [tokens, k]
    counts: torch.Tensor   # int32 [experts]
    tokens: torch.Tensor   # int32 scalar: routed tokens
    loss: torch.Tensor     # fp32 scalar


class MoePlan(NamedTuple):
    rows: torch.Tensor           # int32 [tokens, k]: the row of every slot, -1 = none
    slots: torch.Tensor          # int32 [m]: the slot of every row, -1 = padding
    m_block_group: torch.Tensor  # int32 [m / 128]: the expert of every 128-row block, -1 = none


def _refuse(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _matrix(name: str, t, dtypes=None) -> None:
    _refuse(t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] <= 1), f"{name} must be 2-D with a contiguous last dimension")
    _refuse(dtypes is None or t.dtype in dtypes, f"{name} has the type {t.dtype}")


def _whole(name: str, t, shape, dtype) -> None:
    _refuse(tuple(t.shape) == tuple(shape) and t.dtype == dtype and t.is_contiguous(),
            f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")


def _pitch(t) -> int:
    """Row pitch in elements; of a single row, whose stride torch leaves open, at least the row."""
    return t.stride(-2) if t.shape[-2] > 1 else max(t.stride(-2), t.shape[-1])


def _ptr(t):
    return None if t is None else t.data_ptr()


def _queue(call, device, stream, owned=()):
    """call(stream) with `device` current; `owned` tensors of this call outlive their use on a `stream` that is
    not torch's current one."""
    if device.type != "cuda":
        raise ValueError("the tensors must be on a CUDA device")
    current = torch.cuda.current_stream(device)
    if stream is None:
        stream = current.cuda_stream
    elif stream != current.cuda_stream:
        for t in owned:
            t.record_stream(torch.cuda.ExternalStream(stream, device))
    if device.index == torch.cuda.current_device():
        check(call(stream))
    else:
        with torch.cuda.device(device):
            check(call(stream))


def _same_device(*tensors) -> None:
    devices = {t.device for t in tensors if t is not None}
    _refuse(len(devices) == 1, f"tensors on different devices: {sorted(map(str, devices))}")


def _route_desc(logits, k, renormalize, valid, ids, weights, counts, routed, loss):
    return MoeRouteDesc(logits.data_ptr(), _pitch(logits), logits.shape[0], logits.shape[1], k, _FLOATS[logits.dtype],
                        int(bool(renormalize)), _ptr(valid), ids.data_ptr(), weights.data_ptr(), counts.data_ptr(),
                        routed.data_ptr(), _ptr(loss))


def _check_logits(logits, valid) -> None:
    _matrix("logits", logits, _FLOATS)
    if valid is not None:
        _refuse(valid.dtype in (torch.bool, torch.uint8), "valid must be bool or uint8")
        _whole("valid", valid, (logits.shape[0],), valid.dtype)


def moe_route(logits, k: int, *, renormalize: bool = True, valid=None, stream=None) -> MoeRoute:
    """The k experts with the largest logits (bf16, f16 or fp32 [tokens, experts]) for every token,
    the lower index first among equals; their softmax probabilities as weights (renormalize: divided by their
    sum); the number of slots of every expert; and the balance loss
    experts * sum_e (counts_e / (k N)) * mean_t p_te over the N routed tokens (1 for a uniform router, 0
    for N = 0). A logit of -inf closes that expert to the token; a slot left without an expert has id
    -1 and weight 0. Tokens with valid = False, or with every logit -inf, are not routed, and what
    padding tokens hold is not read. For gradients: moe_route_grad, or torch.ops.kl.moe_route."""
    _check_logits(logits, valid)
    tokens, experts = logits.shape
    _refuse(1 <= k <= experts, f"k must be in [1, {experts}]")
    device = logits.device
    need = ctypes.c_size_t()
    check(lib().kl_moe_route_workspace_size(tokens, experts, ctypes.byref(need)))
    ids = torch.empty((tokens, k), dtype=torch.int32, device=device)
    weights = torch.empty((tokens, k), dtype=torch.float32, device=device)
    counts = torch.empty((experts,), dtype=torch.int32, device=device)
    routed = torch.empty((), dtype=torch.int32, device=device)
    loss = torch.empty((), dtype=torch.float32, device=device)
    work = torch.empty((need.value,), dtype=torch.uint8, device=device) if need.value else None
    _same_device(logits, valid, loss)
    d = _route_desc(logits, k, renormalize, valid, ids, weights, counts, routed, loss)
    out = MoeRoute(ids, weights, counts, routed, loss)
    _queue(lambda s: lib().kl_moe_route(ctypes.byref(d), _ptr(work), need.value, s), device, stream,
           out if work is None else (*out, work))
    return out


def moe_route_grad(logits, route: MoeRoute, dweights=None, dloss=None, *, renormalize: bool = True, valid=None,
                   out=None, stream=None):
    """The gradient of moe_route's logits from those of its weights (fp32 [tokens, k]) and loss (fp32
    scalar); None = 0. `route` is moe_route's result for the same logits, renormalize and valid; its
    counts are constants. `out` may be the logits themselves."""
    _check_logits(logits, valid)
    tokens, experts = logits.shape
    _refuse(route.ids.dim() == 2, "route.ids must be 2-D")
    k = route.ids.shape[1]
    _whole("route.ids", route.ids, (tokens, k), torch.int32)
    _whole("route.weights", route.weights, (tokens, k), torch.float32)
    _whole("route.counts", route.counts, (experts,), torch.int32)
    _whole("route.tokens", route.tokens, (), torch.int32)
    if dweights is not None:
        _whole("dweights", dweights, (tokens, k), torch.float32)
    if dloss is not None:
        _refuse(dloss.numel() == 1 and dloss.dtype == torch.float32, "dloss must be one fp32 value")
    if out is None:
        out = torch.empty((tokens, experts), dtype=logits.dtype, device=logits.device)
    _matrix("out", out, (logits.dtype,))
    _refuse(out.shape == logits.shape, "out must have the logits' shape")
    _same_device(logits, valid, route.ids, route.weights, route.counts, route.tokens, dweights, dloss, out)
    d = _route_desc(logits, k, renormalize, valid, route.ids, route.weights, route.counts, route.tokens, None)
    _queue(lambda s: lib().kl_moe_route_grad(ctypes.byref(d), _ptr(dweights), _ptr(dloss), out.data_ptr(), _pitch(out), s),
           logits.device, stream, (out,))
    return out


def moe_rows(slots: int, experts: int, block: int = 128) -> int:
    """Rows of the grouped layout that any split of `slots` rows over the experts fits."""
    rows = int(lib().kl_moe_rows(int(slots), int(experts), int(block)))
    _refuse(rows >= 0, "slots must not be negative, experts positive, block 128 or 256")
    return rows


def moe_plan(ids, experts: int, *, block: int = 128, stream=None) -> MoePlan:
    """The m-grouped layout of int32 ids [tokens, k] (any other value than 0 .. experts - 1 = no
    expert): the slots sorted by expert, in their order within one, each expert padded to `block`
    rows (256 for gemm_grouped's algo=ALGO_2CTA). Its m = moe_rows(tokens * k, experts, block) rows fit any
    ids, so nothing is read back; blocks behind the last expert have m_block_group -1."""
    _refuse(ids.dim() == 2, "ids must be 2-D")
    _whole("ids", ids, ids.shape, torch.int32)
    tokens, k = ids.shape
    m = moe_rows(tokens * k, experts, block)
    rows = torch.empty((tokens, k), dtype=torch.int32, device=ids.device)
    slots = torch.empty((m,), dtype=torch.int32, device=ids.device)
    groups = torch.empty((m // 128,), dtype=torch.int32, device=ids.device)
    _queue(lambda s: lib().kl_moe_plan(ids.data_ptr(), tokens, k, int(experts), int(block), m, rows.data_ptr(),
                                       slots.data_ptr(), groups.data_ptr(), s), ids.device, stream, (rows, slots, groups))
    return MoePlan(rows, slots, groups)


def _check_plan(rows, slots) -> None:
    _refuse(rows.dim() == 2 and slots.dim() == 1, "rows must be 2-D and slots 1-D, as moe_plan makes them")
    _whole("rows", rows, rows.shape, torch.int32)
    _whole("slots", slots, slots.shape, torch.int32)


def moe_dispatch(x, plan: MoePlan, out=None, *, stream=None):
    """out[row] = x[slots[row] // k]: the tokens' rows (2-D, any type) in the m-grouped layout, every padding row
    zero. Its gradient is moe_combine(dout, rows=plan.rows)."""
    _matrix("x", x)
    _check_plan(plan.rows, plan.slots)
    tokens, k = plan.rows.shape
    m = plan.slots.shape[0]
    _refuse(x.shape[0] == tokens, f"x has {x.shape[0]} rows, the plan {tokens} tokens")
    if out is None:
        out = torch.empty((m, x.shape[1]), dtype=x.dtype, device=x.device)
    _matrix("out", out, (x.dtype,))
    _refuse(out.shape == (m, x.shape[1]), f"out must have the shape {(m, x.shape[1])}")
    _same_device(x, plan.rows, plan.slots, out)
    size = x.element_size()
    _queue(lambda s: lib().kl_moe_dispatch(x.data_ptr(), _pitch(x) * size, tokens, x.shape[1] * size, max(k, 1),
                                           plan.rows.data_ptr(), plan.slots.data_ptr(), m, out.data_ptr(),
                                           _pitch(out) * size, s), x.device, stream, (out,))
    return out


def _rows_of(y, rows, weights):
    """y as a matrix, with (tokens, k), from its rows' indexes or its own [tokens, k, width]."""
    if rows is None:
        _refuse(y.dim() == 3, "without rows, y must be [tokens, k, width]")
        tokens, k = y.shape[:2]
        _refuse(y.is_contiguous(), "without rows, y must be contiguous")
        y = y.view(tokens * k, y.shape[2])
    else:
        _refuse(rows.dim() == 2, "rows must be 2-D")
        _whole("rows", rows, rows.shape, torch.int32)
        tokens, k = rows.shape
    _matrix("y", y, _FLOATS)
    if weights is not None:
        _whole("weights", weights, (tokens, k), torch.float32)
    return y, tokens, k


def moe_combine(y, weights=None, *, rows=None, out=None, stream=None):
    """out[t] = sum_j weights[t, j] * y[rows[t, j]] in fp32, rounded once to y's type (bf16, f16, fp32). y
    is [m, width] with int32 rows [tokens, k] (-1 adds nothing), or [tokens, k, width] without rows.
    weights: fp32 [tokens, k], None = 1."""
    y, tokens, k = _rows_of(y, rows, weights)
    width = y.shape[1]
    if out is None:
        out = torch.empty((tokens, width), dtype=y.dtype, device=y.device)
    _matrix("out", out, (y.dtype,))
    _refuse(out.shape == (tokens, width), f"out must have the shape {(tokens, width)}")
    _same_device(y, rows, weights, out)
    if k == 0:
        return out.zero_()
    _queue(lambda s: lib().kl_moe_combine(y.data_ptr(), _FLOATS[y.dtype], _pitch(y), y.shape[0], _ptr(rows), _ptr(weights),
                                          tokens, k, width, out.data_ptr(), _pitch(out), s), y.device, stream, (out,))
    return out


def moe_combine_grad(dout, y, weights=None, *, rows=None, slots=None, stream=None):
    """(dy, dweights) of moe_combine from dout [tokens, width] of y's type: dy in y's shape and type,
    zero in padding rows; dweights fp32, or None where weights is None. rows and slots are moe_plan's, or
    both None."""
    shape = y.shape
    y, tokens, k = _rows_of(y, rows, weights)
    _refuse((rows is None) == (slots is None), "rows and slots come together")
    if slots is not None:
        _check_plan(rows, slots)
        _refuse(slots.shape[0] == y.shape[0], "slots must have an entry for every row of y")
    _matrix("dout", dout, (y.dtype,))
    _refuse(dout.shape == (tokens, y.shape[1]), f"dout must have the shape {(tokens, y.shape[1])}")
    _same_device(dout, y, weights, rows, slots)
    dy = torch.empty(shape, dtype=y.dtype, device=y.device)
    dweights = None if weights is None else torch.empty((tokens, k), dtype=torch.float32, device=y.device)
    _queue(lambda s: lib().kl_moe_combine_grad(dout.data_ptr(), _pitch(dout), y.data_ptr(), _FLOATS[y.dtype], _pitch(y),
                                               y.shape[0], _ptr(rows), _ptr(slots), _ptr(weights), tokens, max(k, 1),
                                               y.shape[1], dy.data_ptr(), y.shape[1], _ptr(dweights), s),
           y.device, stream, (dy,) if dweights is None else (dy, dweights))
    return dy, dweights


def gemv_int4(x, q, scales, zeros=None, *, group: int = 128, ids=None, out=None, out_dtype=None, stream=None):
    """out = x @ ((q - zeros) * scales).T for few tokens: x bf16 / f16 [tokens, K]; q uint8 [N, K / 2],
    two 4-bit codes a byte, the lower K in the low nibble; scales [N, ceil(K / group)] of x's type or fp32;
    zeros uint8 of the scales' shape (0 .. 127), None = 8. group: 32, 64 or a multiple of 128; K a
    multiple of 32. With int32 ids [tokens, k]: q [E, N, K / 2], scales and zeros [E, N, ...], x [tokens, K]
    or [tokens, k, K], out [tokens, k, N] with expert ids[t, j] (rows of zeros for ids outside 0 .. E - 1). out in
    x's type or fp32; sums in fp32. Up to 32 tokens (16 of one expert) read the weights once."""
    experts = ids is not None
    _refuse(x.dtype in (torch.bfloat16, torch.float16), "x must be bf16 or f16")
    _refuse(q.dtype == torch.uint8 and q.dim() == 2 + experts and q.stride(-1) == 1,
            "q must be uint8 [N, K / 2], or [E, N, K / 2] with ids, its last dimension contiguous")
    n, k = q.shape[-2], q.shape[-1] * 2
    _refuse(group > 0, "group must be positive")
    shape = (*q.shape[:-1], -(-k // group))
    for name, t in (("scales", scales), ("zeros", zeros)):
        _refuse(t is None or (tuple(t.shape) == shape and (t.stride(-1) == 1 or shape[-1] <= 1)),
                f"{name} must have the shape {shape}, its last dimension contiguous")
    _refuse(scales.dtype in (x.dtype, torch.float32), "scales must have x's type or fp32")
    _refuse(zeros is None or zeros.dtype == torch.uint8, "zeros must be uint8")
    per_slot, topk = False, 1
    if experts:
        _refuse(ids.dim() == 2, "ids must be 2-D")
        _whole("ids", ids, ids.shape, torch.int32)
        topk, per_slot = ids.shape[1], x.dim() == 3
        _refuse(x.shape[:-1] == (ids.shape if per_slot else ids.shape[:1]), "x must be [tokens, K] or [tokens, k, K]")
    else:
        _refuse(x.dim() == 2, "x must be [tokens, K]")
    _refuse(x.shape[-1] == k and (x.stride(-1) == 1 or k <= 1), f"x must have {k} contiguous columns")
    _refuse(not per_slot or x.is_contiguous(), "x of [tokens, k, K] must be contiguous")
    tokens = x.shape[0]
    if out is None:
        out = torch.empty((*ids.shape, n) if experts else (tokens, n), dtype=out_dtype or x.dtype, device=x.device)
    _refuse(tuple(out.shape) == ((*ids.shape, n) if experts else (tokens, n)) and out.dtype in (x.dtype, torch.float32),
            "out must be [tokens, N] ([tokens, k, N] with ids) of x's type or fp32")
    _refuse(out.is_contiguous() if experts else out.stride(-1) == 1 or n <= 1, "out must be contiguous in its last dimension")
    _same_device(x, q, scales, zeros, ids, out)
    d = Int4Desc(x.data_ptr(), k if per_slot else _pitch(x), q.data_ptr(), _pitch(q), q.stride(0) if experts else 0,
                 scales.data_ptr(), _pitch(scales), scales.stride(0) if experts else 0,
                 _ptr(zeros), 0 if zeros is None else _pitch(zeros), zeros.stride(0) if experts and zeros is not None else 0,
                 _ptr(ids), q.shape[0] if experts else 0, topk, out.data_ptr(), n if experts else _pitch(out), tokens, n, k, group,
                 _FLOATS[x.dtype], _FLOATS[scales.dtype], _FLOATS[out.dtype], int(per_slot))
    _queue(lambda s: lib().kl_gemv_int4(ctypes.byref(d), s), x.device, stream, (out,))
    return out
