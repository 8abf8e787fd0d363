"""The expert layer's argument checks: nothing here reaches a GPU (host tensors, made-up addresses)."""

import ctypes
import subprocess
import sys

import pytest
import torch

import maia_b200 as kl

P = 0x10000  # an aligned address that no refused call touches


def route_desc(**over):
    d = dict(logits=P, ld_logits=64, tokens=4, experts=64, k=2, logits_type=kl.KL_BF16, renormalize=1, valid=None, ids=P,
             weights=P, counts=P, routed=P, loss=P)
    d.update(over)
    return kl.MoeRouteDesc(**d)


@pytest.mark.parametrize("over, status, what", [
    (dict(experts=0), kl.KL_ERR_NOT_SUPPORTED, "experts"),
    (dict(experts=1025, ld_logits=1025), kl.KL_ERR_NOT_SUPPORTED, "experts"),
    (dict(k=0), kl.KL_ERR_INVALID_ARGUMENT, "k must be"),
    (dict(k=33), kl.KL_ERR_INVALID_ARGUMENT, "k must be"),
    (dict(k=5, experts=4), kl.KL_ERR_INVALID_ARGUMENT, "k must be"),
    (dict(tokens=-1), kl.KL_ERR_INVALID_ARGUMENT, "tokens"),
    (dict(tokens=1 << 26), kl.KL_ERR_INVALID_ARGUMENT, "tokens"),
    (dict(logits_type=kl.KL_E4M3), kl.KL_ERR_NOT_SUPPORTED, "logits must be"),
    (dict(ld_logits=63), kl.KL_ERR_INVALID_ARGUMENT, "pitch"),
    (dict(counts=None), kl.KL_ERR_INVALID_ARGUMENT, "null"),
    (dict(logits=None), kl.KL_ERR_INVALID_ARGUMENT, "null"),
    (dict(tokens=100000), kl.KL_ERR_INVALID_ARGUMENT, "workspace"),
    (dict(logits=P + 1), kl.KL_ERR_INVALID_ARGUMENT, "aligned"),
])
def test_route_refusals(over, status, what):
    d = route_desc(**over)
    with pytest.raises(kl.KlError) as e:
        kl.check(kl.lib().kl_moe_route(ctypes.byref(d), None, 0, None))
    assert e.value.status == status and what in e.value.message


def test_route_null_descriptor():
    assert kl.lib().kl_moe_route(None, None, 0, None) == kl.KL_ERR_INVALID_ARGUMENT
    assert kl.lib().kl_moe_route_grad(None, None, None, None, 0, None) == kl.KL_ERR_INVALID_ARGUMENT
    assert kl.lib().kl_gemv_int4(None, None) == kl.KL_ERR_INVALID_ARGUMENT


def test_route_grad_refusals():
    d = route_desc()
    for args, what in (((None, None, P, 63), "pitch"), ((None, None, None, 64), "null")):
        with pytest.raises(kl.KlError) as e:
            kl.check(kl.lib().kl_moe_route_grad(ctypes.byref(d), *args, None))
        assert what in e.value.message


def test_rows_of_the_layout():
    assert kl.moe_rows(0, 8) == 0
    assert kl.moe_rows(1, 8) == 128
    assert kl.moe_rows(4, 8) == 512            # four slots fill at most four experts' blocks
    assert kl.moe_rows(1000, 8) == (1000 + 8 * 127) // 128 * 128
    assert kl.moe_rows(1000, 8, 256) == (1000 + 8 * 255) // 256 * 256
    for args in ((-1, 8, 128), (1, 0, 128), (1, 8, 64)):
        with pytest.raises(ValueError):
            kl.moe_rows(*args)
    for slots, experts, block in ((0, 8, 128), (1, 8, 128), (77, 5, 256), (1000, 1024, 128)):
        assert kl.moe_rows(slots, experts, block) == kl.lib().kl_moe_rows(slots, experts, block)
    # Never too small: the worst split puts one row into the last block of every expert.
    for slots in range(1, 600, 7):
        for experts in (1, 2, 5):
            holders = min(slots, experts)
            worst = 128 * (holders + (slots - holders) // 128)
            assert kl.moe_rows(slots, experts) >= worst


@pytest.mark.parametrize("over, what", [
    (dict(block=64), "block"), (dict(m=128), "kl_moe_rows"), (dict(m=1000), "multiple"), (dict(k=33), "k in"),
    (dict(tokens=-1), "extents"), (dict(ids=None), "null"), (dict(slots=None), "null"), (dict(experts=0), "experts"),
    (dict(experts=1025), "experts"), (dict(tokens=1 << 30), "rows"),
])
def test_plan_refusals(over, what):
    a = dict(ids=P, tokens=64, k=4, experts=8, block=128, m=1280, rows=P, slots=P, groups=P)
    a.update(over)
    with pytest.raises(kl.KlError) as e:
        kl.check(kl.lib().kl_moe_plan(a["ids"], a["tokens"], a["k"], a["experts"], a["block"], a["m"], a["rows"],
                                      a["slots"], a["groups"], None))
    assert what in e.value.message


def test_row_movers_refusals():
    L = kl.lib()
    for call, what in (
        (lambda: L.kl_moe_dispatch(P, 15, 4, 16, 2, P, P, 128, P, 16, None), "pitch"),
        (lambda: L.kl_moe_dispatch(P, 16, 4, 16, 2, None, P, 128, P, 16, None), "null"),
        (lambda: L.kl_moe_dispatch(P, 16, 4, 16, 0, P, P, 128, P, 16, None), "k in"),
        (lambda: L.kl_moe_combine(P, kl.KL_E4M3, 8, 128, P, P, 4, 2, 8, P, 8, None), "bf16"),
        (lambda: L.kl_moe_combine(P, kl.KL_BF16, 7, 128, P, P, 4, 2, 8, P, 8, None), "pitch"),
        (lambda: L.kl_moe_combine(P, kl.KL_BF16, 8, 9, None, P, 4, 2, 8, P, 8, None), "tokens * k"),
        (lambda: L.kl_moe_combine(P + 1, kl.KL_BF16, 8, 128, P, P, 4, 2, 8, P, 8, None), "aligned"),
        (lambda: L.kl_moe_combine_grad(P, 8, P, kl.KL_F32, 8, 8, None, None, P, 4, 2, 8, P + 2, 8, P, None), "aligned"),
        (lambda: L.kl_moe_combine(None, kl.KL_BF16, 8, 8, None, P, 4, 2, 8, P, 8, None), "null"),
        (lambda: L.kl_moe_combine_grad(P, 8, P, kl.KL_BF16, 8, 8, P, None, P, 4, 2, 8, P, 8, P, None), "together"),
        (lambda: L.kl_moe_combine_grad(P, 7, P, kl.KL_BF16, 8, 8, None, None, P, 4, 2, 8, P, 8, P, None), "pitch"),
        (lambda: L.kl_moe_combine_grad(P, 8, None, kl.KL_BF16, 8, 8, None, None, P, 4, 2, 8, P, 8, P, None), "null"),
    ):
        with pytest.raises(kl.KlError) as e:
            kl.check(call())
        assert e.value.status in (kl.KL_ERR_INVALID_ARGUMENT, kl.KL_ERR_NOT_SUPPORTED) and what in e.value.message


@pytest.mark.parametrize("over, what", [
    (dict(x_type=kl.KL_F32), "x must be"), (dict(scale_type=kl.KL_F16), "scales must"), (dict(out_type=kl.KL_F16), "out must"),
    (dict(group=48), "group"), (dict(group=192), "group"), (dict(group=0), "group"), (dict(k=4080), "multiple of 32"),
    (dict(ldq=2047), "pitch"), (dict(ldx=4095), "pitch"), (dict(ld_scales=31), "pitch"), (dict(zeros=P, ld_zeros=31), "pitch"),
    (dict(ldo=63), "pitch"), (dict(x=P + 2), "aligned"), (dict(q=P + 8), "aligned"), (dict(ldx=4100), "aligned"),
    (dict(ldq=2056), "aligned"), (dict(x=None), "null"), (dict(q=None), "null"), (dict(scales=None), "null"),
    (dict(out=None), "null"), (dict(tokens=-1), "negative"), (dict(tokens=1 << 40), "too large"),
    (dict(ids=P, experts=0, topk=1), "experts"), (dict(ids=P, experts=4, topk=0), "topk"),
    (dict(ids=P, experts=4, topk=2049, tokens=2), "4096"), (dict(ids=P, experts=1025, topk=1), "1024 experts"),
    (dict(ids=P, experts=4, topk=1, stride_q=8), "stride"),
    (dict(scales=P + 1), "aligned"), (dict(out=P + 1), "aligned"), (dict(out=P + 2, out_type=kl.KL_F32), "aligned"),
    (dict(ids=P + 2, experts=1, topk=1), "aligned"),
])
def test_gemv_int4_refusals(over, what):
    d = dict(x=P, ldx=4096, q=P, ldq=2048, scales=P, ld_scales=32, out=P, ldo=64, tokens=1, n=64, k=4096, group=128,
             x_type=kl.KL_BF16, scale_type=kl.KL_BF16, out_type=kl.KL_BF16)
    d.update(over)
    d = kl.Int4Desc(**d)
    with pytest.raises(kl.KlError) as e:
        kl.check(kl.lib().kl_gemv_int4(ctypes.byref(d), None))
    assert what in e.value.message


def test_python_refusals():
    f32, i32 = torch.float32, torch.int32
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    q, s = torch.zeros((8, 32), dtype=torch.uint8), torch.ones((8, 1), dtype=torch.bfloat16)
    plan = kl.MoePlan(torch.zeros((2, 1), dtype=i32), torch.zeros(256, dtype=i32), torch.zeros(2, dtype=i32))
    for call in (
        lambda: kl.moe_route(torch.zeros((2, 4, 4)), 1),
        lambda: kl.moe_route(torch.zeros((2, 4), dtype=torch.float64), 1),
        lambda: kl.moe_route(torch.zeros((4, 2)).T, 1),
        lambda: kl.moe_route(torch.zeros((2, 4)), 5),
        lambda: kl.moe_route(torch.zeros((2, 4)), 1, valid=torch.ones(3, dtype=torch.bool)),
        lambda: kl.moe_route(torch.zeros((2, 4)), 1, valid=torch.ones(2, dtype=i32)),
        lambda: kl.moe_plan(torch.zeros((2, 4), dtype=torch.int64), 4),
        lambda: kl.moe_plan(torch.zeros((4, 2), dtype=i32).T, 4),
        lambda: kl.moe_plan(torch.zeros((2, 4), dtype=i32), 4, block=100),
        lambda: kl.moe_dispatch(torch.zeros((3, 8)), plan),
        lambda: kl.moe_dispatch(torch.zeros((2, 8)), plan, torch.zeros((255, 8))),
        lambda: kl.moe_combine(torch.zeros((2, 8))),
        lambda: kl.moe_combine(torch.zeros((4, 8)), torch.zeros((2, 2), dtype=torch.float64), rows=torch.zeros((2, 2), dtype=i32)),
        lambda: kl.moe_combine(torch.zeros((4, 8), dtype=torch.float64), rows=torch.zeros((2, 2), dtype=i32)),
        lambda: kl.moe_combine_grad(torch.zeros((2, 8)), torch.zeros((4, 8)), rows=torch.zeros((2, 2), dtype=i32)),
        lambda: kl.moe_combine_grad(torch.zeros((2, 7)), torch.zeros((2, 2, 8))),
        lambda: kl.gemv_int4(x.to(f32), q, s, group=64),
        lambda: kl.gemv_int4(x, q, s, group=32),
        lambda: kl.gemv_int4(x, q.to(torch.int8), s, group=64),
        lambda: kl.gemv_int4(x, q, s.to(torch.float16), group=64),
        lambda: kl.gemv_int4(x, q, s, s, group=64),
        lambda: kl.gemv_int4(x[:, :32], q, s, group=64),
        lambda: kl.gemv_int4(x, q, s, group=64, ids=torch.zeros((2, 1), dtype=i32)),
        lambda: kl.gemv_int4(x, q[None], s[None], group=64, ids=torch.zeros((3, 1), dtype=i32)),
        lambda: kl.gemv_int4(x, q, s, group=64, out=torch.zeros((2, 9), dtype=torch.bfloat16)),
        lambda: kl.gemv_int4(x, q, s, group=64),  # host tensors
        lambda: kl.moe_route(torch.zeros((2, 4)), 1),
    ):
        with pytest.raises(ValueError):
            call()


def test_binding_imports_without_torch():
    code = "import sys; sys.modules['torch'] = None; import maia_b200 as kl; print(kl.lib().kl_moe_rows(1, 1, 128))"
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, check=True)
    assert out.stdout.strip() == "128"


def test_fake_tensor_shapes():
    import maia_b200.torch_ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        logits = torch.empty((10, 8), dtype=torch.bfloat16)
        ids, weights, counts, tokens, loss = torch.ops.kl.moe_route(logits, 2)
        assert ids.shape == weights.shape == (10, 2) and ids.dtype == torch.int32 and weights.dtype == torch.float32
        assert counts.shape == (8,) and tokens.shape == loss.shape == ()
        rows, slots, groups = torch.ops.kl.moe_plan(ids, 8)
        m = kl.moe_rows(20, 8)
        assert rows.shape == (10, 2) and slots.shape == (m,) and groups.shape == (m // 128,)
        a = torch.ops.kl.moe_dispatch(torch.empty((10, 64), dtype=torch.float16), rows, slots)
        assert a.shape == (m, 64) and a.dtype == torch.float16
        assert torch.ops.kl.moe_combine(a, weights, rows, slots).shape == (10, 64)
        assert torch.ops.kl.moe_combine(torch.empty((10, 2, 32)), weights).shape == (10, 32)
        x, q, s = torch.empty((3, 64), dtype=torch.bfloat16), torch.empty((40, 32), dtype=torch.uint8), torch.empty((40, 1))
        assert torch.ops.kl.gemv_int4(x, q, s, None, 64).shape == (3, 40)
        ids = torch.empty((3, 2), dtype=torch.int32)
        y = torch.ops.kl.gemv_int4(x, q[None], s[None], None, 64, ids, torch.float32)
        assert y.shape == (3, 2, 40) and y.dtype == torch.float32
