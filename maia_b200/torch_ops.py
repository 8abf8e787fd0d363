"""PyTorch operators over the C ABI: torch.ops.kl.gemm, torch.ops.kl.gemm_fp8,
torch.ops.kl.gemm_block_scaled and torch.ops.kl.gemm_grouped; around the last the expert layer's
torch.ops.kl.moe_route, moe_plan, moe_dispatch and moe_combine, with gradients, and torch.ops.kl.gemv_int4.

Registered with torch.library so they compose with the rest of a PyTorch program (fake tensors
for shape inference, the dispatcher, torch.compile graphs that call them as opaque ops). The work
is the library's own kernels, launched on the tensors' current CUDA stream.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ALGO_1CTA, ALGO_2CTA, ALGO_AUTO, experts as _experts, gemm as _kl_gemm, gemm_grouped as _kl_gemm_grouped


@torch.library.custom_op("kl::gemm", mutates_args=())
def gemm(a: torch.Tensor, b: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16, alpha: float = 1.0) -> torch.Tensor:
    """alpha * a @ b.T for bf16 a [M, K] and b [N, K] (K contiguous), out bf16 or fp32."""
    if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        raise TypeError("kl::gemm takes bf16 operands (use kl::gemm_fp8 for e4m3)")
    out = torch.empty((a.shape[0], b.shape[0]), dtype=out_dtype, device=a.device)
    return _kl_gemm(a, b, out, alpha=alpha, algo=ALGO_AUTO)


@gemm.register_fake
def _(a, b, out_dtype=torch.bfloat16, alpha=1.0):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=out_dtype)


@torch.library.custom_op("kl::gemm_fp8", mutates_args=())
def gemm_fp8(a: torch.Tensor, b: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor) -> torch.Tensor:
    """(a @ b.T) * scale_a * scale_b for e4m3 a [M, K], b [N, K] and fp32 scalar scales; bf16 out."""
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn:
        raise TypeError("kl::gemm_fp8 takes float8_e4m3fn operands")
    out = torch.empty((a.shape[0], b.shape[0]), dtype=torch.bfloat16, device=a.device)
    return _kl_gemm(a, b, out, scale_a=scale_a.float().contiguous(), scale_b=scale_b.float().contiguous(),
                    algo=ALGO_AUTO)


@gemm_fp8.register_fake
def _(a, b, scale_a, scale_b):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=torch.bfloat16)


@torch.library.custom_op("kl::gemm_block_scaled", mutates_args=())
def gemm_block_scaled(a: torch.Tensor, b: torch.Tensor, sfa: torch.Tensor, sfb: torch.Tensor, scale_vec: int = 32,
                      out_dtype: torch.dtype = torch.bfloat16, scale_a: Optional[torch.Tensor] = None,
                      scale_b: Optional[torch.Tensor] = None, fp6: str = "") -> torch.Tensor:
    """Block-scaled a @ b.T: a [M, K] and b [N, K] in float8_e4m3fn / float8_e5m2 (MXFP8, scale_vec
    32) or float4_e2m1fn_x2 ([M, K/2]; MXFP4 with scale_vec 32, NVFP4 with scale_vec 16), or with
    fp6 = "e3m2" / "e2m3" uint8 packed fp6 ([M, 3K/4], MXFP6); sfa / sfb the uint8 scales in the
    blocked layout of maia_b200.pack_block_scales, optional fp32 scalar per-tensor scales; bf16 or
    fp32 out."""
    out = torch.empty((a.shape[0], b.shape[0]), dtype=out_dtype, device=a.device)
    return _kl_gemm(a, b, out, sfa=sfa, sfb=sfb, scale_vec=scale_vec,
                    scale_a=None if scale_a is None else scale_a.float().contiguous(),
                    scale_b=None if scale_b is None else scale_b.float().contiguous(), algo=ALGO_AUTO,
                    ab_type=fp6 or None)


@gemm_block_scaled.register_fake
def _(a, b, sfa, sfb, scale_vec=32, out_dtype=torch.bfloat16, scale_a=None, scale_b=None, fp6=""):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=out_dtype)


@torch.library.custom_op("kl::gemm_grouped", mutates_args=())
def gemm_grouped(a: torch.Tensor, b: torch.Tensor, m_block_group: torch.Tensor,
                 out_dtype: torch.dtype = torch.bfloat16, pairs: bool = False) -> torch.Tensor:
    """m-grouped a @ b[g].T (mixture-of-experts layout): a [M, K] with the groups' rows back to back
    (each group padded to 128 rows, or 256 with pairs=True for the CTA-pair kernel), b [G, N, K],
    m_block_group int32 [ceil(M / 128)] naming each 128-row block's group (-1 = padding)."""
    out = torch.empty((a.shape[0], b.shape[1]), dtype=out_dtype, device=a.device)
    return _kl_gemm_grouped(a, b, m_block_group, out, algo=ALGO_2CTA if pairs else ALGO_1CTA)


@gemm_grouped.register_fake
def _(a, b, m_block_group, out_dtype=torch.bfloat16, pairs=False):
    return a.new_empty((a.shape[0], b.shape[1]), dtype=out_dtype)


@torch.library.custom_op("kl::moe_route", mutates_args=())
def moe_route(logits: torch.Tensor, k: int, renormalize: bool = True, valid: Optional[torch.Tensor] = None
              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(ids, weights, counts, routed tokens, balance loss) of logits [tokens, experts]: maia_b200.moe_route.
    Differentiable in weights and loss; the choice of experts and the counts are constants."""
    return tuple(_experts.moe_route(logits, k, renormalize=renormalize, valid=valid))


@moe_route.register_fake
def _(logits, k, renormalize=True, valid=None):
    tokens, experts = logits.shape
    whole = dict(dtype=torch.int32)
    return (logits.new_empty((tokens, k), **whole), logits.new_empty((tokens, k), dtype=torch.float32),
            logits.new_empty((experts,), **whole), logits.new_empty((), **whole), logits.new_empty((), dtype=torch.float32))


@torch.library.custom_op("kl::moe_route_grad", mutates_args=())
def moe_route_grad(logits: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, counts: torch.Tensor, tokens: torch.Tensor,
                   dweights: Optional[torch.Tensor], dloss: Optional[torch.Tensor], renormalize: bool,
                   valid: Optional[torch.Tensor]) -> torch.Tensor:
    """The gradient of kl::moe_route's logits: maia_b200.moe_route_grad."""
    route = _experts.MoeRoute(ids, weights, counts, tokens, None)
    return _experts.moe_route_grad(logits, route, dweights, dloss, renormalize=renormalize, valid=valid)


@moe_route_grad.register_fake
def _(logits, ids, weights, counts, tokens, dweights, dloss, renormalize, valid):
    return logits.new_empty(logits.shape)


def _route_context(ctx, inputs, output):
    logits, _, ctx.renormalize, valid = inputs
    ids, weights, counts, tokens, _ = output
    ctx.save_for_backward(logits, ids, weights, counts, tokens, valid)
    ctx.mark_non_differentiable(ids, counts, tokens)


def _route_backward(ctx, _ids, dweights, _counts, _tokens, dloss):
    logits, ids, weights, counts, tokens, valid = ctx.saved_tensors
    dlogits = torch.ops.kl.moe_route_grad(logits, ids, weights, counts, tokens,
                                          None if dweights is None else dweights.contiguous(),
                                          None if dloss is None else dloss.contiguous(), ctx.renormalize, valid)
    return dlogits, None, None, None


moe_route.register_autograd(_route_backward, setup_context=_route_context)


@torch.library.custom_op("kl::moe_plan", mutates_args=())
def moe_plan(ids: torch.Tensor, experts: int, block: int = 128) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(rows, slots, m_block_group) of int32 ids [tokens, k]: maia_b200.moe_plan."""
    return tuple(_experts.moe_plan(ids, experts, block=block))


@moe_plan.register_fake
def _(ids, experts, block=128):
    m = _experts.moe_rows(ids.shape[0] * ids.shape[1], experts, block)
    return ids.new_empty(ids.shape), ids.new_empty((m,)), ids.new_empty((m // 128,))


@torch.library.custom_op("kl::moe_dispatch", mutates_args=())
def moe_dispatch(x: torch.Tensor, rows: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """x's rows in the m-grouped layout of kl::moe_plan's rows and slots: maia_b200.moe_dispatch."""
    return _experts.moe_dispatch(x, _experts.MoePlan(rows, slots, None))


@moe_dispatch.register_fake
def _(x, rows, slots):
    return x.new_empty((slots.shape[0], x.shape[1]))


def _dispatch_context(ctx, inputs, output):
    ctx.save_for_backward(inputs[1])


def _dispatch_backward(ctx, da):
    (rows,) = ctx.saved_tensors
    return torch.ops.kl.moe_combine(da.contiguous(), None, rows, None), None, None


moe_dispatch.register_autograd(_dispatch_backward, setup_context=_dispatch_context)


@torch.library.custom_op("kl::moe_combine", mutates_args=())
def moe_combine(y: torch.Tensor, weights: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The weighted sum of each token's rows of y: maia_b200.moe_combine. Differentiable in y and weights; with rows
    that takes kl::moe_plan's slots too."""
    return _experts.moe_combine(y, weights, rows=rows)


@moe_combine.register_fake
def _(y, weights=None, rows=None, slots=None):
    return y.new_empty((y.shape[0] if rows is None else rows.shape[0], y.shape[-1]))


@torch.library.custom_op("kl::moe_combine_grad", mutates_args=())
def moe_combine_grad(dout: torch.Tensor, y: torch.Tensor, weights: torch.Tensor, rows: Optional[torch.Tensor],
                     slots: Optional[torch.Tensor], want_dy: bool = True, want_dweights: bool = True
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gradients of kl::moe_combine's y and weights: maia_b200.moe_combine_grad. What is not wanted is empty."""
    both = _experts.moe_combine_grad(dout, y, weights, rows=rows, slots=slots, want_dy=want_dy, want_dweights=want_dweights)
    return tuple(t.new_empty((0,)) if g is None else g for g, t in zip(both, (y, weights)))


@moe_combine_grad.register_fake
def _(dout, y, weights, rows, slots, want_dy=True, want_dweights=True):
    return y.new_empty(y.shape if want_dy else (0,)), weights.new_empty(weights.shape if want_dweights else (0,))


def _combine_context(ctx, inputs, output):
    y, weights, rows, slots = inputs
    ctx.shape = y.shape
    ctx.save_for_backward(None if weights is None else y, weights, rows, slots)


def _combine_backward(ctx, dout):
    y, weights, rows, slots = ctx.saved_tensors
    if rows is not None and slots is None:
        raise RuntimeError("kl::moe_combine with rows needs kl::moe_plan's slots for its gradient")
    if weights is None:  # a copy of dout for every slot
        if rows is None:
            return dout[:, None].expand(ctx.shape), None, None, None
        return torch.ops.kl.moe_dispatch(dout.contiguous(), rows, slots), None, None, None
    want_dy, want_dweights = ctx.needs_input_grad[:2]
    dy, dweights = torch.ops.kl.moe_combine_grad(dout.contiguous(), y, weights, rows, slots, want_dy, want_dweights)
    return dy if want_dy else None, dweights if want_dweights else None, None, None


moe_combine.register_autograd(_combine_backward, setup_context=_combine_context)


@torch.library.custom_op("kl::gemv_int4", mutates_args=())
def gemv_int4(x: torch.Tensor, q: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, group: int = 128,
              ids: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Products of few tokens with 4-bit weights, of one matrix or of the experts that `ids` names:
    maia_b200.gemv_int4. For inference: no gradient."""
    return _experts.gemv_int4(x, q, scales, zeros, group=group, ids=ids, out_dtype=out_dtype)


@gemv_int4.register_fake
def _(x, q, scales, zeros=None, group=128, ids=None, out_dtype=None):
    shape = (x.shape[0], q.shape[0]) if ids is None else (*ids.shape, q.shape[1])
    return x.new_empty(shape, dtype=out_dtype or x.dtype)
