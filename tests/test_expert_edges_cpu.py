"""The expert layer's refusals and host-side rules beside those of test_experts_cpu.py; nothing here reaches a GPU."""

import ctypes

import pytest

import maia_b200 as kl
from test_experts_cpu import P, route_desc


def refused(status, what):
    with pytest.raises(kl.KlError) as e:
        kl.check(status)
    assert e.value.status == kl.KL_ERR_INVALID_ARGUMENT and what in e.value.message, e.value.message


@pytest.mark.parametrize("field", ["ids", "weights", "counts", "routed", "loss"])
@pytest.mark.parametrize("off", [1, 2])
def test_route_misaligned_arrays(field, off):
    refused(kl.lib().kl_moe_route(ctypes.byref(route_desc(**{field: P + off})), None, 0, None), "4-byte aligned")
    if field != "loss":  # not the gradient's
        refused(kl.lib().kl_moe_route_grad(ctypes.byref(route_desc(**{field: P + off})), P, P, P, 64, None), "4-byte aligned")


def test_route_grad_misaligned_gradients():
    for dweights, dloss in ((P + 2, P), (P, P + 1), (P + 1, None), (None, P + 2)):
        refused(kl.lib().kl_moe_route_grad(ctypes.byref(route_desc()), dweights, dloss, P, 64, None), "4-byte aligned")


@pytest.mark.parametrize("at", range(4))
def test_row_movers_misaligned_arrays(at):
    L, w = kl.lib(), [P + 2 * (i == at) for i in range(4)]
    refused(L.kl_moe_plan(w[0], 64, 4, 8, 128, 1280, w[1], w[2], w[3], None), "4-byte aligned")
    refused(L.kl_moe_combine_grad(P, 8, P, kl.KL_BF16, 8, 8, w[0], w[1], w[2], 4, 2, 8, P, 8, w[3], None), "4-byte aligned")
    if at < 2:
        refused(L.kl_moe_dispatch(P, 16, 4, 16, 2, w[0], w[1], 128, P, 16, None), "4-byte aligned")
        refused(L.kl_moe_combine(P, kl.KL_BF16, 8, 128, w[0], w[1], 4, 2, 8, P, 8, None), "4-byte aligned")


def test_host_tensors_are_refused_on_any_stream():
    import torch

    x, q, s = torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros((8, 32), dtype=torch.uint8), torch.ones((8, 1), dtype=torch.bfloat16)
    for call in (lambda: kl.moe_route(torch.zeros((2, 4)), 1, stream=16), lambda: kl.gemv_int4(x, q, s, group=64, stream=0),
                 lambda: kl.moe_combine(torch.zeros((2, 2, 8)), stream=16)):
        with pytest.raises(ValueError):
            call()


def test_a_single_row_has_no_pitch():
    """Whatever buffer one token's row was cut from, its pitch is its own length: no alignment is asked of the buffer's."""
    import torch

    from maia_b200.experts import _pitch

    base = torch.empty((6, 4100))
    assert _pitch(base[:1, :4096]) == 4096 and _pitch(base[:2, :4096]) == 4100 and _pitch(base[::5][:1]) == 4100
    assert _pitch(base[:0, :64]) == 64 and _pitch(torch.empty((3, 1, 48))[..., :32]) == 32


def test_combine_grad_of_one_output():
    """dy or dweights may be left out, not both; what is left out is not checked, what is read is."""
    L = kl.lib()
    refused(L.kl_moe_combine_grad(P, 8, P, kl.KL_BF16, 8, 8, None, None, P, 4, 2, 8, None, 8, None, None), "null")
    refused(L.kl_moe_combine_grad(P, 8, None, kl.KL_BF16, 8, 8, None, None, P, 4, 2, 8, None, 8, P, None), "null")
    refused(L.kl_moe_combine_grad(None, 8, P, kl.KL_BF16, 8, 8, None, None, P, 4, 2, 8, None, 0, P, None), "null")
    assert L.kl_moe_combine_grad(None, 8, None, kl.KL_BF16, 8, 128, P, P, P, 0, 2, 8, None, 0, P, None) == kl.KL_OK  # no tokens


def test_gemv_int4_refusal_names_a_way():
    """Too many pairs: the message names what takes them, which no other product of the library does with 4-bit codes."""
    d = kl.Int4Desc(x=P, ldx=4096, q=P, ldq=2048, scales=P, ld_scales=32, out=P, ldo=64, tokens=2049, n=64, k=4096, group=128,
                    ids=P, experts=4, topk=2, stride_q=64 * 2048, stride_scales=64 * 32,
                    x_type=kl.KL_BF16, scale_type=kl.KL_BF16, out_type=kl.KL_BF16)
    with pytest.raises(kl.KlError) as e:
        kl.check(kl.lib().kl_gemv_int4(ctypes.byref(d), None))
    assert "calls of some of them" in e.value.message and "GEMM" not in e.value.message


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dloss", [None, 2.0])
def test_the_oracles_gradient_against_differences(renormalize, dloss):
    """expert_oracle.route_grad, which the kernel's gradient is held to, against central differences of expert_oracle.route:
    closed experts, fewer open ones than k, a row with none, padding. The choice is held by gaps between the logits."""
    import math

    import torch

    import expert_oracle as oracle

    tokens, experts, k, h = 6, 9, 3, 1e-5
    rng = lambda i: torch.Generator().manual_seed(i)  # noqa: E731
    x = torch.stack([torch.randperm(experts, generator=rng(i)).double() * 0.3 for i in range(tokens)])
    x[1, ::2] = -math.inf
    x[2, 2:] = -math.inf                       # two open experts for three slots
    x[3] = -math.inf
    valid = torch.tensor([True, True, True, True, False, True])
    dw = torch.randn((tokens, k), generator=rng(9)).double()

    def value(z):
        ids, w, _, _, loss, _ = oracle.route(z, k, renormalize, valid)
        return (w * dw)[ids >= 0].sum().item() + (dloss or 0.0) * loss

    got = oracle.route_grad(x, k, dw, dloss, renormalize, valid)
    assert (got[3:5] == 0).all()
    for t in range(tokens):
        for e in range(experts):
            up, down = x.clone(), x.clone()
            up[t, e] += h
            down[t, e] -= h
            want = (value(up) - value(down)) / (2 * h)
            # A third derivative below 50 by h^2 / 6, and values below 50 rounded to 2^-53 each over 2 h.
            assert abs(got[t, e].item() - want) <= 50 * h * h / 6 + 64 * 50 * 2.0 ** -53 / h, (t, e)
