"""The expert layer and the 4-bit products at the ends of what their documentation allows, against the definitions in
64 bits (tests/expert_oracle.py). u = 2^-24 is half a step of fp32, relative to the value."""

import math

import pytest
import torch

import expert_oracle as oracle
import maia_b200 as kl

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
F64 = torch.float64


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, tol, what=""):
    off = (got.detach().cpu().to(F64) - want.cpu()).abs()
    assert got.shape == want.shape and bool((off <= tol.cpu()).all()), f"{what}: off by {(off / tol.cpu().clamp(min=1e-300)).max().item():.2f} of the tolerance"


def product_tol(x, w, want, dtype, groups):
    """An element of x enters whole, so only fp32 sums of exact products are off, relative to the products' sizes: 16
    steps within a group's product, 4 roundings for its scale and its digits, a sum a group, 16 warps and 8 blocks."""
    size = x.to(F64).abs() @ w.abs().transpose(-1, -2)
    return size * (groups + 48) * U + want.abs() * HALF[dtype] * 1.001 + torch.finfo(dtype).smallest_normal * HALF[dtype] * 2


# ------------------------------------------------------------------------------------ 4-bit products


@pytest.mark.parametrize("tokens", [1, 2, 3, 16])
@pytest.mark.parametrize("group", [2 ** 31 - 128, 2 ** 31, 2 ** 32, 2 ** 32 + 128, 2 ** 40, 2 ** 62])
def test_gemv_int4_group_longer_than_32_bits(cuda, tokens, group):
    """One scale for a row, asked for by a group length that 32 bits do not hold."""
    n, k = 40, 1056
    q = torch.randint(0, 256, (n, k // 2), generator=gen(1), dtype=torch.uint8).to(cuda)
    s = (torch.rand((n, 1), generator=gen(2)) * 0.02 + 0.001).bfloat16().to(cuda)
    z = torch.randint(0, 16, (n, 1), generator=gen(3), dtype=torch.uint8).to(cuda)
    x = torch.randn((tokens, k), generator=gen(4)).bfloat16().to(cuda)
    got = kl.gemv_int4(x, q, s, z, group=group)
    assert torch.equal(got, kl.gemv_int4(x, q, s, z, group=1152))
    ids = torch.tensor([[0, 1]] * tokens, dtype=torch.int32, device=cuda)
    by_expert = kl.gemv_int4(x, torch.stack([q, q]), torch.stack([s, s]), torch.stack([z, z]), group=group, ids=ids)
    want = x.cpu().to(F64) @ oracle.int4_weights(q, s, z, 1152).T
    # Two forms of one product: each rounds fp32 sums of it once to bf16.
    slack = product_tol(x.cpu(), oracle.int4_weights(q, s, z, 1152), want, torch.bfloat16, 9) + 2.0 ** -21 * x.abs().max().item() * oracle.int4_weights(q, s, z, 1152).abs().sum(1)
    within(got, want, slack)
    for j in range(2):
        within(by_expert[:, j], want, slack)


# ------------------------------------------------------------------------------------ streams

PENDING = 100_000_000  # cycles that a stream is kept busy: 50 ms


def calls(cuda):
    """name -> (a call on a stream, fresh tensors that it reads)."""
    tokens, experts, k, width = 3000, 64, 4, 264
    logits = torch.randn((tokens, experts), generator=gen(1)).to(cuda)
    x = torch.randn((tokens, width), generator=gen(2)).bfloat16().to(cuda)
    route = kl.moe_route(logits, k)
    plan = kl.moe_plan(route.ids, experts)
    y = kl.moe_dispatch(x, plan)
    dw = torch.randn((tokens, k), generator=gen(3)).to(cuda)
    q = torch.randint(0, 256, (4096, 256), generator=gen(4), dtype=torch.uint8).to(cuda)
    s = torch.ones((4096, 4), device=cuda).bfloat16()
    v = torch.randn((300, 512), generator=gen(5)).bfloat16().to(cuda)
    some = torch.randint(-1, 2, (300, 2), generator=gen(6), dtype=torch.int32).to(cuda)
    return {
        "route": (lambda st, t: kl.moe_route(t, k, stream=st), logits),
        "route_grad": (lambda st, t: kl.moe_route_grad(t, route, dw, route.loss, stream=st), logits),
        "plan": (lambda st, t: kl.moe_plan(t, experts, stream=st), route.ids),
        "dispatch": (lambda st, t: kl.moe_dispatch(t, plan, stream=st), x),
        "combine": (lambda st, t: kl.moe_combine(t, dw, rows=plan.rows, stream=st), y),
        "combine_grad": (lambda st, t: kl.moe_combine_grad(t, y, dw, rows=plan.rows, slots=plan.slots, stream=st), x),
        "gemv": (lambda st, t: kl.gemv_int4(t, q, s, stream=st), v),
        "gemv_by_expert": (lambda st, t: kl.gemv_int4(v, q.view(2, 2048, 256), s.view(2, 2048, 4), ids=t, stream=st), some),
    }


def several(result):
    return [t for t in (result if isinstance(result, tuple) else (result,)) if t is not None]


NAMES = ["route", "route_grad", "plan", "dispatch", "combine", "combine_grad", "gemv", "gemv_by_expert"]


@pytest.mark.parametrize("name", NAMES)
def test_memory_that_the_current_stream_still_uses(cuda, name):
    """A call on another stream takes none of the blocks that were just given back while work queued on the
    current stream still reads them, its workspace's among them."""
    call, t = calls(cuda)[name]
    want = [r.clone() for r in several(call(None, t))]
    need = kl.experts._route_workspace(3000, 64)
    sizes = [r.numel() * r.element_size() for r in want] + [need]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(2):
        freed = [torch.full((size,), 7, dtype=torch.uint8, device=cuda) for size in sizes for _ in range(2)]
        torch.cuda._sleep(PENDING)
        copies = [f.clone() for f in freed]
        del freed
        got = several(call(side.cuda_stream, t))
        side.synchronize()
        same = [g.clone() for g in got]
        torch.cuda.synchronize()
        assert all((c == 7).all() for c in copies)
        assert all(torch.equal(a, b) for a, b in zip(same, want))


@pytest.mark.parametrize("name", [n for n in NAMES if n not in ("plan", "gemv_by_expert")])
def test_inputs_dropped_while_another_stream_reads_them(cuda, name):
    call, t = calls(cuda)[name]
    want = [r.clone() for r in several(call(None, t))]
    side = torch.cuda.Stream()
    mine = t.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(PENDING)
    got = several(call(side.cuda_stream, mine))
    del mine
    over = [torch.full_like(t, 3) for _ in range(4)]  # would take the block that was given back
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and len(over) == 4


@pytest.mark.parametrize("name", NAMES)
def test_outputs_dropped_while_the_current_stream_reads_them(cuda, name):
    """What a call on another stream returns may be used on the current stream and dropped there."""
    call, t = calls(cuda)[name]
    want = [r.clone() for r in several(call(None, t))]
    side, zero = torch.cuda.Stream(), torch.zeros_like(t)
    torch.cuda.synchronize()
    got = several(call(side.cuda_stream, t))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(PENDING)
    copies = [g.clone() for g in got]
    del got
    call(side.cuda_stream, zero)  # would write where the first results lay
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(copies, want))


def test_the_default_stream_by_its_handle(cuda):
    x = torch.randn((3000, 64), generator=gen(1)).to(cuda)
    want = kl.moe_route(x, 4)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = kl.moe_route(x, 4, stream=0)
        torch.cuda.default_stream().synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()


def test_nothing_to_add_on_another_stream(cuda):
    """No slots at all: the zeros are written on the stream that was asked for."""
    side = torch.cuda.Stream()
    out = torch.full((50, 64), 5.0, device=cuda)
    torch.cuda.synchronize()
    torch.cuda._sleep(PENDING)
    kl.moe_combine(torch.empty((50, 0, 64), device=cuda), out=out, stream=side.cuda_stream)
    side.synchronize()
    with torch.cuda.stream(side):
        zero = (out == 0).all()
        side.synchronize()
    assert bool(zero)
    torch.cuda.synchronize()


def products(cuda):
    """name -> a call on a stream of the package's GEMMs and quantisers that make their own outputs."""
    x = torch.randn((512, 1024), generator=gen(1)).bfloat16().to(cuda)
    w = torch.randn((2, 768, 1024), generator=gen(2)).bfloat16().to(cuda)
    blocks = torch.tensor([0, 1, 1, 0], dtype=torch.int32, device=cuda)
    scales = torch.randint(100, 140, (512, 32), generator=gen(3), dtype=torch.uint8).to(cuda)
    return {
        "gemm": lambda st: kl.gemm(x, w[0], stream=st),
        "gemm_grouped": lambda st: kl.gemm_grouped(x, w, blocks, stream=st),
        "pack_block_scales": lambda st: kl.pack_block_scales(scales, 1024, stream=st),
        "mx_quantize": lambda st: kl.mx_quantize(x, stream=st),
        "nv_quantize": lambda st: kl.nv_quantize(x, stream=st),
    }


@pytest.mark.parametrize("name", ["gemm", "gemm_grouped", "pack_block_scales", "mx_quantize", "nv_quantize"])
def test_outputs_of_products_on_another_stream(cuda, name):
    """Likewise for the calls around the GEMMs that make their outputs: none lies where the current stream still reads."""
    call = products(cuda)[name]
    bits = lambda t: t.contiguous().view(torch.uint8).clone()  # noqa: E731
    want = [bits(r) for r in several(call(None))]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(2):
        freed = [torch.full((w.numel(),), 7, dtype=torch.uint8, device=cuda) for w in want for _ in range(2)]
        torch.cuda._sleep(PENDING)
        copies = [f.clone() for f in freed]
        del freed
        got = several(call(side.cuda_stream))
        side.synchronize()
        with torch.cuda.stream(side):
            same = [bits(g) for g in got]
        torch.cuda.synchronize()
        assert all((c == 7).all() for c in copies)
        assert all(torch.equal(a, b) for a, b in zip(same, want))
