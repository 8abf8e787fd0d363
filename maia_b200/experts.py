"""Mixture-of-experts routing around gemm_grouped, and decode products with 4-bit weights.

    r = moe_route(logits, k)                        # experts and weights of every token, counts, balance loss
    plan = moe_plan(r.ids, experts)                 # rows of the m-grouped layout
    a = moe_dispatch(x, plan)
    y = gemm_grouped(a, w, plan.m_block_group)      # one matrix per expert
    out = moe_combine(y, r.weights, rows=plan.rows)

For a few tokens, without a layout: y = gemv_int4(x, q, scales, ids=r.ids); out = moe_combine(y, r.weights).
Every call is queued on the tensors' current CUDA stream and allocates only its outputs (moe_route a workspace too),
through torch. With `stream`, a raw handle, it runs as with that stream current: the caller orders the two streams, as
for torch's own calls, and keeps the handle valid while tensors of the call live. No counterpart in the reference
(kernel_lib has no GEMM and no routing).
"""

from __future__ import annotations

import ctypes
import struct
from functools import lru_cache
from typing import NamedTuple

import torch

from . import Int4Desc, KL_BF16, KL_F16, KL_F32, KL_OK, MoeRouteDesc, _on_stream, check, lib

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


# torch's own cheap forms of current_stream(device).cuda_stream and current_device(): a decode step makes
# a handful of calls of a few microseconds each.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _packer(desc):
    """desc(*fields) as bytes, at a quarter of the structure's cost."""
    kinds = {ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int32: "i"}
    packed = struct.Struct("@" + "".join(kinds[kind] for _, kind in desc._fields_))
    assert packed.size == ctypes.sizeof(desc)
    return packed.pack


_pack_route, _pack_int4 = _packer(MoeRouteDesc), _packer(Int4Desc)


def _refuse(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _matrix(name: str, t, dtypes=None) -> None:
    if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1 and t.shape[0] > 0):  # torch leaves an empty tensor's strides open
        raise ValueError(f"{name} must be 2-D with a contiguous last dimension")
    if dtypes is not None and t.dtype not in dtypes:
        raise ValueError(f"{name} has the type {t.dtype}")


def _whole(name: str, t, shape, dtype) -> None:
    if t.shape != shape or t.dtype is not dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")


def _pitch(t) -> int:
    """Row pitch in elements; of a single row, which has none, the row."""
    shape = t.shape
    return t.stride(-2) if shape[-2] > 1 else shape[-1]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _device(first, *others) -> int:
    """The one CUDA device of the tensors (None = not given)."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError("the tensors must be on one CUDA device")
    if index < 0:
        raise ValueError("the tensors must be on a CUDA device")
    return index


def _queue(device: int, fn, *args) -> None:
    """fn(*args, the device's current stream) with `device` current."""
    if device == _current_device():
        status = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(device))
    if status != KL_OK:
        check(status)


@lru_cache(maxsize=4096)
def _route_workspace(tokens: int, experts: int) -> int:
    need = ctypes.c_size_t()
    check(lib().kl_moe_route_workspace_size(tokens, experts, ctypes.byref(need)))
    return need.value


def _route_desc(logits, k, renormalize, valid, ids, weights, counts, routed, loss):
    return _pack_route(logits.data_ptr(), _pitch(logits), logits.shape[0], logits.shape[1], k, _FLOATS[logits.dtype],
                       bool(renormalize), _ptr(valid) or 0, ids.data_ptr(), weights.data_ptr(), counts.data_ptr(),
                       routed.data_ptr(), _ptr(loss) or 0)


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
    if stream is not None:
        return _on_stream(stream, (logits, valid), lambda: moe_route(logits, k, renormalize=renormalize, valid=valid))
    _check_logits(logits, valid)
    tokens, experts = logits.shape
    if not 1 <= k <= experts:
        raise ValueError(f"k must be in [1, {experts}]")
    device = _device(logits, valid)
    ids = logits.new_empty((tokens, k), dtype=torch.int32)
    weights = logits.new_empty((tokens, k), dtype=torch.float32)
    counts = logits.new_empty((experts,), dtype=torch.int32)
    routed = logits.new_empty((), dtype=torch.int32)
    loss = logits.new_empty((), dtype=torch.float32)
    size = _route_workspace(tokens, experts)
    work = logits.new_empty((size,), dtype=torch.uint8) if size else None
    d = _route_desc(logits, k, renormalize, valid, ids, weights, counts, routed, loss)
    _queue(device, lib().kl_moe_route, d, _ptr(work), size)
    return MoeRoute(ids, weights, counts, routed, loss)


def moe_route_grad(logits, route: MoeRoute, dweights=None, dloss=None, *, renormalize: bool = True, valid=None,
                   out=None, stream=None):
    """The gradient of moe_route's logits from those of its weights (fp32 [tokens, k]) and loss (fp32
    scalar); None = 0. `route` is moe_route's result for the same logits, renormalize and valid; its
    counts are constants. `out` may be the logits themselves."""
    if stream is not None:
        return _on_stream(stream, (logits, *route, dweights, dloss, valid, out),
                          lambda: moe_route_grad(logits, route, dweights, dloss, renormalize=renormalize, valid=valid, out=out))
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
        out = logits.new_empty((tokens, experts))
    _matrix("out", out, (logits.dtype,))
    _refuse(out.shape == logits.shape, "out must have the logits' shape")
    device = _device(logits, valid, route.ids, route.weights, route.counts, route.tokens, dweights, dloss, out)
    d = _route_desc(logits, k, renormalize, valid, route.ids, route.weights, route.counts, route.tokens, None)
    _queue(device, lib().kl_moe_route_grad, d, _ptr(dweights), _ptr(dloss), out.data_ptr(), _pitch(out))
    return out


def moe_rows(slots: int, experts: int, block: int = 128) -> int:
    """Rows of the grouped layout that any split of `slots` rows over the experts fits (kl_moe_rows)."""
    if slots < 0 or experts < 1 or block not in (128, 256):
        raise ValueError("slots must not be negative, experts positive, block 128 or 256")
    return (slots + min(slots, experts) * (block - 1)) // block * block


def moe_plan(ids, experts: int, *, block: int = 128, stream=None) -> MoePlan:
    """The m-grouped layout of int32 ids [tokens, k] (any other value than 0 .. experts - 1 = no
    expert): the slots sorted by expert, in their order within one, each expert padded to `block`
    rows (256 for gemm_grouped's algo=ALGO_2CTA). Its m = moe_rows(tokens * k, experts, block) rows fit any
    ids, so nothing is read back; blocks behind the last expert have m_block_group -1."""
    if stream is not None:
        return _on_stream(stream, (ids,), lambda: moe_plan(ids, experts, block=block))
    _refuse(ids.dim() == 2, "ids must be 2-D")
    _whole("ids", ids, ids.shape, torch.int32)
    tokens, k = ids.shape
    m = moe_rows(tokens * k, experts, block)
    device = _device(ids)
    plan = MoePlan(torch.empty_like(ids), ids.new_empty((m,)), ids.new_empty((m // 128,)))
    if k == 0:
        return plan
    _queue(device, lib().kl_moe_plan, ids.data_ptr(), tokens, k, experts, block, m, plan.rows.data_ptr(),
           plan.slots.data_ptr(), plan.m_block_group.data_ptr())
    return plan


def _check_plan(rows, slots) -> None:
    if (rows.dim() != 2 or slots.dim() != 1 or rows.dtype is not torch.int32 or slots.dtype is not torch.int32
            or not rows.is_contiguous() or not slots.is_contiguous()):
        raise ValueError("rows must be 2-D and slots 1-D, contiguous int32, as moe_plan makes them")


def moe_dispatch(x, plan: MoePlan, out=None, *, stream=None):
    """out[row] = x[slots[row] // k]: the tokens' rows (2-D, any type) in the m-grouped layout, every padding row
    zero. Its gradient is moe_combine(dout, rows=plan.rows)."""
    if stream is not None:
        return _on_stream(stream, (x, plan.rows, plan.slots, out), lambda: moe_dispatch(x, plan, out))
    rows, slots = plan.rows, plan.slots
    _matrix("x", x)
    _check_plan(rows, slots)
    tokens, k = rows.shape
    m, width, size = slots.shape[0], x.shape[1], x.element_size()
    if x.shape[0] != tokens:
        raise ValueError(f"x has {x.shape[0]} rows, the plan {tokens} tokens")
    if out is None:
        out = x.new_empty((m, width))
    else:
        _matrix("out", out, (x.dtype,))
        _refuse(out.shape == (m, width), f"out must have the shape {(m, width)}")
    device = _device(x, rows, slots, out)
    if k == 0:
        return out.zero_()
    _queue(device, lib().kl_moe_dispatch, x.data_ptr(), _pitch(x) * size, tokens, width * size, k, rows.data_ptr(), slots.data_ptr(), m, out.data_ptr(), _pitch(out) * size)
    return out


def _rows_of(y, rows, weights):
    """(tokens, k, rows of y, width, row pitch) from y's row indexes, or its own [tokens, k, width]."""
    if rows is None:
        if y.dim() != 3 or not y.is_contiguous() or y.dtype not in _FLOATS:
            raise ValueError("without rows, y must be contiguous bf16, f16 or fp32 [tokens, k, width]")
        tokens, k, width = y.shape
        m, pitch = tokens * k, width
    else:
        _refuse(rows.dim() == 2, "rows must be 2-D")
        _whole("rows", rows, rows.shape, torch.int32)
        _matrix("y", y, _FLOATS)
        tokens, k = rows.shape
        m, width = y.shape
        pitch = _pitch(y)
    if weights is not None:
        _whole("weights", weights, (tokens, k), torch.float32)
    return tokens, k, m, width, pitch


def moe_combine(y, weights=None, *, rows=None, out=None, stream=None):
    """out[t] = sum_j weights[t, j] * y[rows[t, j]] in fp32, rounded once to y's type (bf16, f16, fp32). y
    is [m, width] with int32 rows [tokens, k] (-1 adds nothing), or [tokens, k, width] without rows.
    weights: fp32 [tokens, k], None = 1."""
    if stream is not None:
        return _on_stream(stream, (y, weights, rows, out), lambda: moe_combine(y, weights, rows=rows, out=out))
    tokens, k, m, width, pitch = _rows_of(y, rows, weights)
    if out is None:
        out = y.new_empty((tokens, width))
    else:
        _matrix("out", out, (y.dtype,))
        _refuse(out.shape == (tokens, width), f"out must have the shape {(tokens, width)}")
    device = _device(y, rows, weights, out)
    if k == 0:
        return out.zero_()
    _queue(device, lib().kl_moe_combine, y.data_ptr(), _FLOATS[y.dtype], pitch, m, _ptr(rows), _ptr(weights),
           tokens, k, width, out.data_ptr(), _pitch(out))
    return out


def moe_combine_grad(dout, y, weights=None, *, rows=None, slots=None, want_dy=True, want_dweights=True, stream=None):
    """(dy, dweights) of moe_combine from dout [tokens, width] of y's type: dy in y's shape and type,
    zero in padding rows; dweights fp32, or None where weights is None. rows and slots are moe_plan's, or
    both None. What is not wanted is None and not computed; without dweights y is not read."""
    if stream is not None:
        return _on_stream(stream, (dout, y, weights, rows, slots),
                          lambda: moe_combine_grad(dout, y, weights, rows=rows, slots=slots, want_dy=want_dy,
                                                   want_dweights=want_dweights))
    tokens, k, m, width, pitch = _rows_of(y, rows, weights)
    _refuse((rows is None) == (slots is None), "rows and slots come together")
    if slots is not None:
        _whole("slots", slots, (m,), torch.int32)
    _matrix("dout", dout, (y.dtype,))
    if dout.shape != (tokens, width):
        raise ValueError(f"dout must have the shape {(tokens, width)}")
    device = _device(dout, y, weights, rows, slots)
    dweights = torch.empty_like(weights) if want_dweights and weights is not None else None
    if k == 0:
        return y.new_zeros(y.shape) if want_dy else None, dweights
    dy = y.new_empty(y.shape) if want_dy else None
    if dy is None and dweights is None:
        return None, None
    _queue(device, lib().kl_moe_combine_grad, dout.data_ptr(), _pitch(dout), y.data_ptr(), _FLOATS[y.dtype], pitch, m, _ptr(rows), _ptr(slots), _ptr(weights), tokens, k,
           width, _ptr(dy), width, _ptr(dweights))
    return dy, dweights


def gemv_int4(x, q, scales, zeros=None, *, group: int = 128, ids=None, out=None, out_dtype=None, stream=None):
    """out = x @ ((q - zeros) * scales).T for few tokens: x bf16 / f16 [tokens, K]; q uint8 [N, K / 2],
    two 4-bit codes a byte, the lower K in the low nibble; scales [N, ceil(K / group)] of x's type or fp32;
    zeros uint8 of the scales' shape, None = 8. group: 32, 64 or a multiple of 128; K a
    multiple of 32. With int32 ids [tokens, k]: q [E, N, K / 2], scales and zeros [E, N, ...], x [tokens, K]
    or [tokens, k, K], out [tokens, k, N] with expert ids[t, j] (rows of zeros for ids outside 0 .. E - 1;
    at most 4096 ids, 1024 experts). out in x's type or fp32. x enters with all its bits, sums are exact or fp32; a NaN
    or infinity makes its row NaN or infinite. K up to 65536. Up to 16 tokens of a matrix read its weights once (8 where
    K > 22528, 2 where K > 28672, by ids a little earlier). With ids the number goes by the average of ids to an expert,
    rounded up to 1, 2, 8 or 16; an expert with more reads its weights several times."""
    if stream is not None:
        return _on_stream(stream, (x, q, scales, zeros, ids, out),
                          lambda: gemv_int4(x, q, scales, zeros, group=group, ids=ids, out=out, out_dtype=out_dtype))
    dtype, bits = x.dtype, x.dim()
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError("x must be bf16 or f16")
    if q.dtype is not torch.uint8 or q.dim() != (2 if ids is None else 3) or (q.stride(-1) != 1 and q.shape[-1] > 1):
        raise ValueError("q must be uint8 [N, K / 2], or [E, N, K / 2] with ids, its last dimension contiguous")
    _refuse(group > 0, "group must be positive")
    n, k = q.shape[-2], q.shape[-1] * 2
    groups = -(-k // group)
    shape = (n, groups) if ids is None else (q.shape[0], n, groups)
    if scales.shape != shape or (scales.stride(-1) != 1 and groups > 1) or (scales.dtype is not dtype and scales.dtype is not torch.float32):
        raise ValueError(f"scales must have the shape {shape}, its last dimension contiguous, and x's type or fp32")
    if zeros is not None and (zeros.shape != shape or (zeros.stride(-1) != 1 and groups > 1) or zeros.dtype is not torch.uint8):
        raise ValueError(f"zeros must be uint8 of the shape {shape}, its last dimension contiguous")
    tokens = x.shape[0]
    if ids is None:
        if bits != 2 or x.shape[1] != k or (x.stride(1) != 1 and k > 1):
            raise ValueError(f"x must be [tokens, {k}], its last dimension contiguous")
        result, topk, per_slot, ldx = (tokens, n), 1, False, _pitch(x)
    else:
        _refuse(ids.dim() == 2, "ids must be 2-D")
        _whole("ids", ids, ids.shape, torch.int32)
        topk, per_slot = ids.shape[1], bits == 3
        if x.shape != ((*ids.shape, k) if per_slot else (ids.shape[0], k)) or (x.stride(-1) != 1 and k > 1):
            raise ValueError(f"x must be [tokens, {k}] or [tokens, k, {k}], its last dimension contiguous")
        _refuse(not per_slot or x.is_contiguous(), "x of [tokens, k, K] must be contiguous")
        result, ldx = (tokens, topk, n), k if per_slot else _pitch(x)
    if out is None:
        out_dtype = out_dtype or dtype
        out = x.new_empty(result) if out_dtype is dtype else x.new_empty(result, dtype=out_dtype)
    elif out.shape != result:
        raise ValueError(f"out must have the shape {result}")
    else:
        _refuse(out.stride(-1) == 1 or n <= 1 if ids is None else out.is_contiguous(), "out must be contiguous in its last dimension")
    if out.dtype is not dtype and out.dtype is not torch.float32:
        raise ValueError("out must have x's type or fp32")
    device = _device(x, q, scales, zeros, ids, out)
    if topk == 0:
        return out
    one = ids is None
    zero_fields = (0, 0, 0) if zeros is None else (zeros.data_ptr(), _pitch(zeros), 0 if one else zeros.stride(0))
    d = _pack_int4(x.data_ptr(), ldx, q.data_ptr(), _pitch(q), 0 if one else q.stride(0),
                   scales.data_ptr(), _pitch(scales), 0 if one else scales.stride(0), *zero_fields,
                   0 if one else ids.data_ptr(), 0 if one else q.shape[0], topk, out.data_ptr(), _pitch(out) if one else n,
                   tokens, n, k, group, _FLOATS[dtype], _FLOATS[scales.dtype], _FLOATS[out.dtype], per_slot)
    _queue(device, lib().kl_gemv_int4, d)
    return out
