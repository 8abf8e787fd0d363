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


def product_tol(x, w, want, dtype):
    """An element of x enters whole, so only fp32 sums are off, relative to the products' sizes. With up to two tokens
    x is taken apart into signed digits, whose sizes add up to at most three times its own (every digit below the first is at
    most half of its base). A sum meets at most one rounding for every 32 elements and scale, and 32 for
    a group's 8 products of 16, its scale, the digits, 16 warps and 8 blocks; what is a tensor core's own cuts at 2 U."""
    size = x.to(F64).abs() @ w.abs().transpose(-1, -2)
    k = x.shape[-1]
    return 3 * size * (k / 32 + 32) * U + want.abs() * HALF[dtype] * 1.001 + torch.finfo(dtype).smallest_normal * HALF[dtype] * 2


# ------------------------------------------------------------------------------------ routing


@pytest.mark.parametrize("experts", [4, 64, 300])
def test_route_weights_far_below_the_largest(cuda, experts):
    """Chosen experts whose probabilities go down through fp32's subnormals: each keeps its own bits."""
    tokens, k = 40, 3
    x = torch.full((tokens, experts), -300.0)
    x[:, 0] = torch.randn(tokens, generator=gen(1))
    x[:, 2] = x[:, 0] - torch.linspace(1, 102, tokens)
    x[:, 3] = x[:, 2] - 0.5
    p = torch.softmax(x.to(F64), 1)[:, [0, 2, 3]]
    reach = (x[:, :1] - x[:, [0, 2, 3]]).to(F64)
    for renormalize in (False, True):
        r = kl.moe_route(x.to(cuda), k, renormalize=renormalize)
        assert r.ids.cpu().tolist() == [[0, 2, 3]] * tokens
        want = p / p.sum(1, keepdim=True) if renormalize else p
        # The difference's rounding (|l - max| U), expf's two steps, sum, reciprocal and product; the last step of a subnormal.
        within(r.weights, want, want * (reach + 16) * U + 2.0 ** -149, f"renormalize {renormalize}")


# ------------------------------------------------------------------------------------ offsets behind 2^31


def test_rows_behind_2_to_the_31_elements(cuda):
    """Dispatch, combine and its gradient on matrices of more than 2^31 elements."""
    tokens, width = 67000, 32776
    x = torch.empty((tokens, width), dtype=torch.bfloat16, device=cuda)
    x.copy_(torch.arange(width, device=cuda)[None] % 64)
    x[:, 0] = (torch.arange(tokens, device=cuda) % 256).bfloat16()
    x[:, 1] = (torch.arange(tokens, device=cuda) // 256).bfloat16()  # both exact: every row has its own
    ids = torch.randint(0, 3, (tokens, 1), generator=gen(1), dtype=torch.int32).to(cuda)
    plan = kl.moe_plan(ids, 3)
    a = kl.moe_dispatch(x, plan)
    assert a.numel() > 2 ** 31
    slots = plan.slots.long()
    live = slots >= 0
    assert torch.equal(a[live, :2], x[slots[live], :2]) and not a[~live].any()
    assert torch.equal(a[-200:], torch.where(live[-200:, None], x[slots[-200:].clamp(min=0)], 0))
    w = torch.full((tokens, 1), 0.5, device=cuda)
    out = kl.moe_combine(a, w, rows=plan.rows)
    assert torch.equal(out[-200:], x[-200:] / 2) and torch.equal(out[:, :2], x[:, :2] / 2)
    del out
    dy, dw = kl.moe_combine_grad(x, a, w, rows=plan.rows, slots=plan.slots)
    assert torch.equal(dy[live, :2], x[slots[live], :2] / 2) and not dy[~live].any()
    tail = x[-200:].double().square().sum(1)
    within(dw[-200:, 0], tail, tail * (width / 256 + 32) * U)


def test_routing_behind_2_to_the_31_logits(cuda):
    tokens, experts, k = 2 ** 21 + 300, 1024, 2
    x = torch.empty((tokens, experts), dtype=torch.bfloat16, device=cuda).uniform_(-1, 1)
    assert x.numel() > 2 ** 31
    x[-300:, 7], x[-300:, 1000] = 3.0, 2.5
    r = kl.moe_route(x, k)
    assert r.tokens.item() == tokens and r.counts.sum().item() == tokens * k
    assert (r.ids[-300:] == torch.tensor([7, 1000], device=cuda)).all()
    g = kl.moe_route_grad(x, r, torch.ones_like(r.weights) * torch.tensor([1.0, -1.0], device=cuda))
    w = r.weights[-300:].double()
    want = 2 * w[:, 0] * w[:, 1]      # w0 (1 - (w0 - w1)) = 2 w0 w1
    within(g[-300:, 7], want, want * (HALF[torch.bfloat16] * 1.001 + 64 * U) + 2.0 ** -24)


# ------------------------------------------------------------------------------------ plans of several sizes


def test_plans_of_many_and_few_experts_in_one_graph(cuda):
    many, few = (torch.randint(-1, e, (700, 3), generator=gen(e), dtype=torch.int32).to(cuda) for e in (1024, 300))
    want = (*kl.moe_plan(many, 1024), *kl.moe_plan(few, 300))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = (*kl.moe_plan(many, 1024), *kl.moe_plan(few, 300))
    kl.moe_plan(few, 300)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_plans_of_many_and_few_experts_from_two_threads(cuda):
    """Every call keeps the shared memory that it needs, whatever another thread plans."""
    import threading

    sizes = (1024, 300)
    ids = [torch.randint(-1, e, (700, 3), generator=gen(e), dtype=torch.int32).to(cuda) for e in sizes]
    want = [kl.moe_plan(i, e) for i, e in zip(ids, sizes)]
    torch.cuda.synchronize()
    wrong = []

    def plan(at):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(2000):
                    got = kl.moe_plan(ids[at], sizes[at])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[at])):
                    wrong.append("another plan")
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=plan, args=(at,)) for at in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


# ------------------------------------------------------------------------------------ combine's gradients, one by one


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens, k, width", [(1, 1, 1), (37, 3, 1001), (70, 8, 264)])
@pytest.mark.parametrize("grouped", [True, False])
def test_combine_gradients_one_by_one(cuda, dtype, tokens, k, width, grouped):
    """Each gradient by itself is what both calls give, bit for bit, in the C call and through autograd, and the one that is
    not asked for reads nothing of its own."""
    import maia_b200.torch_ops  # noqa: F401

    rows = slots = None
    y = torch.randn((tokens, k, width), generator=gen(1)).to(dtype).to(cuda)
    if grouped:
        plan = kl.moe_plan(torch.randint(-1, 5, (tokens, k), generator=gen(2), dtype=torch.int32).to(cuda), 5)
        rows, slots = plan.rows, plan.slots
        y = torch.randn((slots.shape[0], width), generator=gen(3)).to(dtype).to(cuda)
    w = torch.rand((tokens, k), generator=gen(4)).to(cuda)
    dout = torch.randn((tokens, width), generator=gen(5)).to(dtype).to(cuda)
    dy, dw = kl.moe_combine_grad(dout, y, w, rows=rows, slots=slots)
    only, none = kl.moe_combine_grad(dout, torch.full_like(y, math.nan), w, rows=rows, slots=slots, want_dweights=False)
    assert none is None and torch.equal(only, dy)
    none, only = kl.moe_combine_grad(dout, y, w, rows=rows, slots=slots, want_dy=False)
    assert none is None and torch.equal(only, dw)
    assert kl.moe_combine_grad(dout, y, w, rows=rows, slots=slots, want_dy=False, want_dweights=False) == (None, None)
    plain, _ = kl.moe_combine_grad(dout, y, rows=rows, slots=slots)
    for needs_y, needs_w in ((True, True), (True, False), (False, True)):
        leaves = [y.clone().requires_grad_(needs_y), w.clone().requires_grad_(needs_w)]
        torch.ops.kl.moe_combine(*leaves, rows, slots).backward(dout)
        assert torch.equal(leaves[0].grad, dy) if needs_y else leaves[0].grad is None
        assert torch.equal(leaves[1].grad, dw) if needs_w else leaves[1].grad is None
    leaf = y.clone().requires_grad_()
    torch.ops.kl.moe_combine(leaf, None, rows, slots).backward(dout)
    assert torch.equal(leaf.grad, plain)


def test_unweighted_combine_keeps_nothing_of_its_rows(cuda):
    """y itself is not needed for its gradient without weights: it may be written over before the backward pass."""
    import maia_b200.torch_ops  # noqa: F401

    leaf = torch.randn((5, 2, 16), device=cuda, requires_grad=True)
    y = leaf * 1
    out = torch.ops.kl.moe_combine(y)
    y.detach().zero_()
    out.backward(torch.ones_like(out))
    assert (leaf.grad == 1).all()


# ------------------------------------------------------------------------------------ nothing to do


def test_no_tokens_through_torch_ops(cuda):
    """A batch without tokens, forward and backward from a broadcast gradient, whose strides torch leaves at 0."""
    import maia_b200.torch_ops  # noqa: F401

    logits = torch.empty((0, 8), device=cuda, requires_grad=True)
    x = torch.empty((0, 64), device=cuda, requires_grad=True)
    ids, weights, _, _, loss = torch.ops.kl.moe_route(logits, 2)
    rows, slots, _ = torch.ops.kl.moe_plan(ids, 8)
    y = torch.ops.kl.moe_dispatch(x, rows, slots)
    (torch.ops.kl.moe_combine(y, weights, rows, slots).sum() + loss + y.sum()).backward()
    assert x.grad.shape == (0, 64) and logits.grad.shape == (0, 8)
    y = torch.empty((0, 2, 64), device=cuda, requires_grad=True)
    torch.ops.kl.moe_combine(y).sum().backward()
    assert y.grad.shape == y.shape


@pytest.mark.parametrize("tokens", [0, 3])
def test_no_slots_at_all(cuda, tokens):
    """k = 0 through plan, dispatch, combine, their gradients and the products by expert: empty or zero everywhere."""
    import maia_b200.torch_ops  # noqa: F401

    ids = torch.empty((tokens, 0), dtype=torch.int32, device=cuda)
    plan = kl.moe_plan(ids, 8)
    assert plan.rows.shape == (tokens, 0) and plan.slots.shape == (0,) and plan.m_block_group.shape == (0,)
    x = torch.randn((tokens, 64), device=cuda)
    a = kl.moe_dispatch(x, plan)
    assert a.shape == (0, 64)
    w = torch.empty((tokens, 0), device=cuda)
    padding = torch.randn((256, 64), device=cuda)       # a layout with padding alone
    slots = torch.full((256,), -1, dtype=torch.int32, device=cuda)
    out = torch.full((256, 64), 5.0, device=cuda)
    assert kl.moe_dispatch(x, kl.MoePlan(ids, slots, None), out) is out and (out == 0).all()
    for weights in (w, None):
        for y, rows, at in ((a, plan.rows, plan.slots), (padding, ids, slots), (torch.empty((tokens, 0, 64), device=cuda), None, None)):
            assert torch.equal(kl.moe_combine(y, weights, rows=rows), torch.zeros_like(x))
            dy, dw = kl.moe_combine_grad(x, y, weights, rows=rows, slots=at)
            assert torch.equal(dy, torch.zeros_like(y)) and (dw is None if weights is None else dw.shape == (tokens, 0))
            leaf = y.clone().requires_grad_()
            torch.ops.kl.moe_combine(leaf, weights, rows, at).sum().backward()
            assert torch.equal(leaf.grad, torch.zeros_like(y))
    leaf = x.clone().requires_grad_()
    torch.ops.kl.moe_dispatch(leaf, plan.rows, plan.slots).sum().backward()
    assert torch.equal(leaf.grad, torch.zeros_like(x))
    q = torch.zeros((4, 16, 32), dtype=torch.uint8, device=cuda)
    s = torch.ones((4, 16, 2), dtype=torch.bfloat16, device=cuda)
    for v in (x.bfloat16(), torch.empty((tokens, 0, 64), dtype=torch.bfloat16, device=cuda)):
        assert kl.gemv_int4(v, q, s, group=32, ids=ids).shape == (tokens, 0, 16)
    torch.cuda.synchronize()


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
    slack = product_tol(x.cpu(), oracle.int4_weights(q, s, z, 1152), want, torch.bfloat16)
    within(got, want, slack)
    for j in range(2):
        within(by_expert[:, j], want, slack)



def check_products(x, q, s, z, group, cuda, what=""):
    """Every row of x by itself, in pairs and all together, dense and by expert, into x's type and fp32."""
    w = oracle.int4_weights(q, s, z, group)
    want = x.to(F64) @ w.T
    xd, tokens = x.to(cuda), x.shape[0]
    on = [None if t is None else t.to(cuda) for t in (q, s, z)]
    for step in (1, 2, tokens):
        for dtype in (x.dtype, torch.float32):
            got = torch.cat([kl.gemv_int4(xd[i:i + step], *on, group=group, out_dtype=dtype) for i in range(0, tokens, step)])
            within(got, want, product_tol(x, w, want, dtype), f"{what}, {step} tokens into {dtype}")
    two = [None if t is None else torch.stack([t, t]) for t in on]
    ids = torch.arange(tokens, dtype=torch.int32, device=cuda)[:, None] % 2
    for i in range(0, tokens, 4):  # two tokens to an expert
        got = kl.gemv_int4(xd[i:i + 4], *two, group=group, ids=ids[i:i + 4], out_dtype=torch.float32)[:, 0]
        within(got, want[i:i + 4], product_tol(x[i:i + 4], w, want[i:i + 4], torch.float32), f"{what}, by expert")


@pytest.mark.parametrize("dtype, outlier", [(torch.bfloat16, 1000.0), (torch.bfloat16, 1e30), (torch.float16, 1000.0),
                                            (torch.float16, 4096.0), (torch.float16, 60000.0)])
@pytest.mark.parametrize("group, zeros", [(32, True), (64, True), (64, False), (128, False), (256, True)])
def test_gemv_int4_small_beside_large(cuda, dtype, outlier, group, zeros):
    """An element far above its neighbours that meets a code equal to the zero point: the neighbours alone make the
    result, and keep every bit."""
    n, k, tokens = 40, 1056, 8
    q = torch.randint(0, 256, (n, k // 2), generator=gen(group), dtype=torch.uint8)
    s = (torch.rand((n, -(-k // group)), generator=gen(2)) * 0.02 + 0.001).to(dtype)
    z = torch.randint(0, 256 if group == 64 else 16, s.shape, generator=gen(3), dtype=torch.uint8) % 16 if zeros else None
    x = (torch.randn((tokens, k), generator=gen(4)) * 0.01).to(dtype)
    codes = torch.stack([q % 16, q // 16], -1).flatten(-2)
    for i in range(0, k, 128):
        at = i + (37 * i // 128) % min(128, k - i)
        x[i // 128 % tokens:, at] = outlier    # some tokens' and not others'
        codes[:, at] = 8 if z is None else z[:, at // group]
    q = codes[:, 0::2] | codes[:, 1::2] << 4
    check_products(x, q, s, z, group, cuda, f"outlier {outlier}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("high_zeros", [False, True])
def test_gemv_int4_values_of_all_sizes(cuda, dtype, group, high_zeros):
    """Elements spread over the exponents of the type, zero points up to 255: each counts with all its bits, alone (the
    others' codes at the zero point) and together."""
    n, k, tokens = 72, 640, 6
    low, high = (-60, 60) if dtype is torch.bfloat16 else (-24, 15)
    x = (torch.randn((tokens, k), generator=gen(1)).clamp(-1.9, 1.9) * 2.0 ** torch.randint(low, high, (tokens, k), generator=gen(2))).to(dtype)
    z = torch.randint(0, 16, (n, k // group), generator=gen(3), dtype=torch.uint8)
    codes = torch.randint(0, 16, (n, k), generator=gen(4), dtype=torch.uint8)
    at = torch.arange(k) // group
    codes[8:] = z[8:][:, at]
    codes[torch.arange(8, n), torch.randint(0, k, (n - 8,), generator=gen(5))] = 3
    if high_zeros:
        z[4:8] = torch.randint(120, 256, z[4:8].shape, generator=gen(6), dtype=torch.uint8)
    q = codes[:, 0::2] | codes[:, 1::2] << 4
    s = torch.ones(z.shape).to(dtype)
    # f16 holds no sum of these: what it would round to infinity is left to fp32's comparison.
    if dtype is torch.float16:
        s = s / 4096
        x = x.clamp(-2048, 2048)
    check_products(x, q, s, z, group, cuda)


@pytest.mark.parametrize("tokens", [1, 2])
def test_gemv_int4_small_beside_large_over_a_cluster(cuda, tokens):
    """K cut over blocks, tiles shared between warps, some 128s with and most without a large element."""
    n, k, group = 16 * 160 + 5, 24576, 64
    g = torch.Generator("cuda").manual_seed(1)
    codes = torch.randint(0, 16, (n, k), generator=g, device=cuda, dtype=torch.uint8)
    s = (torch.rand((n, k // group), generator=g, device=cuda) * 0.02 + 0.001).bfloat16()
    x = (torch.randn((tokens, k), generator=g, device=cuda) * 0.01).bfloat16()
    for i in range(5, k, 1408):
        x[i % tokens, i] = 2.0 ** 40
        codes[:, i] = 8
    w = (codes.double() - 8) * s.double().repeat_interleave(group, 1)
    want = x.double() @ w.T
    got = kl.gemv_int4(x, codes[:, 0::2] | codes[:, 1::2] << 4, s, group=group, out_dtype=torch.float32)
    within(got, want, product_tol(x, w, want, torch.float32))


def test_gemv_int4_bad_rows_beside_rests(cuda):
    """A token with a NaN or an infinity beside one whose elements leave rests: the second is not touched."""
    n, k = 40, 512
    q = torch.randint(0, 256, (n, k // 2), generator=gen(1), dtype=torch.uint8).to(cuda)
    s = torch.ones((n, 4), dtype=torch.bfloat16, device=cuda)
    x = (torch.randn((2, k), generator=gen(2)) * 1e-9).bfloat16().to(cuda)
    x[1, ::128] = 4.0
    alone = kl.gemv_int4(x, q, s, out_dtype=torch.float32)
    for bad in (math.nan, math.inf):
        x[0, 3] = bad
        got = kl.gemv_int4(x, q, s, out_dtype=torch.float32)
        assert not got[0].isfinite().any() and torch.equal(got[1], alone[1])



def test_one_row_of_a_wider_buffer(cuda):
    """One token, one weight row: cut from buffers whose pitch fits no load, with a base that does."""
    k, n = 256, 24
    x = torch.randn((4, k + 4), generator=gen(1)).bfloat16()
    q = torch.randint(0, 256, (n, k // 2 + 3), generator=gen(2), dtype=torch.uint8)
    s = torch.ones((n, 2), dtype=torch.bfloat16)
    xd, qd, sd = x.to(cuda)[:1, :k], q.to(cuda)[:1, :k // 2], s.to(cuda)[:1]
    w = oracle.int4_weights(q[:1, :k // 2], s[:1], None, 128)
    want = x[:1, :k].to(F64) @ w.T
    within(kl.gemv_int4(xd, qd, sd), want, product_tol(x[:1, :k], w, want, torch.bfloat16))
    got = kl.gemv_int4(xd, qd[None], sd[None], ids=torch.zeros((1, 1), dtype=torch.int32, device=cuda))
    within(got[0], want, product_tol(x[:1, :k], w, want, torch.bfloat16))
    logits = torch.randn((2, 67), generator=gen(3)).to(cuda)
    r, whole = kl.moe_route(logits[:1, :64], 4), kl.moe_route(logits[:1, :64].contiguous(), 4)
    assert all(torch.equal(a, b) for a, b in zip(r, whole))
    dw = torch.randn((1, 4), generator=gen(4)).to(cuda)
    assert torch.equal(kl.moe_route_grad(logits[:1, :64], r, dw), kl.moe_route_grad(logits[:1, :64].contiguous(), r, dw))



@pytest.mark.parametrize("tokens", [1, 20])
def test_gemv_int4_weights_behind_2_to_the_31_bytes(cuda, tokens):
    """The last of the experts lies 2 GB behind the first, its scales 2^27 elements."""
    experts, n, k, group = 130, 16384, 2048, 32
    q = torch.empty((experts, n, k // 2), dtype=torch.uint8, device=cuda).random_(0, 256)
    s = torch.empty((experts, n, k // group), dtype=torch.bfloat16, device=cuda).uniform_(0.001, 0.02)
    ids = torch.tensor([[experts - 1, 0]], dtype=torch.int32, device=cuda).repeat(tokens, 1)
    x = torch.randn((tokens, k), generator=gen(1)).bfloat16().to(cuda)
    got = kl.gemv_int4(x, q, s, group=group, ids=ids, out_dtype=torch.float32)
    for j, e in enumerate((experts - 1, 0)):
        w = (torch.stack([q[e] & 15, q[e] >> 4], -1).flatten(-2).double() - 8) * s[e].double().repeat_interleave(group, 1)
        want = x.double() @ w.T
        within(got[:, j], want, product_tol(x, w, want, torch.float32), f"expert {e}")


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
