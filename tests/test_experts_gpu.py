"""The expert layer on the GPU against its definitions in 64 bits (tests/expert_oracle.py).

Tolerances count roundings. u = 2^-24 is half a step of fp32, relative to the value."""

import math
import pathlib
import subprocess
import sys

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


def close(got, want, tol, what=""):
    """|got - want| <= tol elementwise, NaN and infinities in the same places."""
    got, want = got.detach().cpu().to(F64), want.to(F64)
    assert got.shape == want.shape, what
    same = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~same & ~torch.isnan(want)], want[~same & ~torch.isnan(want)]), what
    off = (got - want).abs()[same]
    tol = torch.as_tensor(tol, dtype=F64).expand(want.shape)[same]
    assert bool((off <= tol).all()), f"{what}: off by {off.max().item():.3e}, {(off / tol.clamp(min=1e-300)).max().item():.2f} of the tolerance"


def prob_tol(logits):
    """Relative error of a probability or normalised weight: the difference l - max is off by half a step (a
    relative error of exp of |l - max| u), expf by 2 steps = 4u, the sum of at most 1024 positive
    terms by 8 NV + 5 roundings (a lane's own, then shuffles) <= 40 u, reciprocal and product 4 u, for numerator and sum."""
    x = logits.detach().cpu().to(F64)
    x = x[torch.isfinite(x)]
    reach = (x.max() - x.min()).item() if x.numel() else 0.0
    return (2 * min(reach, 110.0) + 64) * U


# ------------------------------------------------------------------------------------ routing

def check_route(r, logits, k, renormalize, valid=None):
    ids, weights, counts, routed, loss, probs = oracle.route(logits, k, renormalize, valid)
    assert torch.equal(r.ids.cpu(), ids)
    assert torch.equal(r.counts.cpu(), counts)
    assert r.tokens.item() == routed
    tol = prob_tol(logits)
    close(r.weights, weights, weights.abs().nan_to_num() * tol + 1e-37, "weights")
    # The loss adds positive terms: tokens of a group one after another, 8 warps, up to 296 blocks, experts.
    steps = logits.shape[0] / 8 + 8 + 296 + logits.shape[1] / 256 + 40
    close(r.loss, torch.tensor(loss), (0.0 if math.isnan(loss) else abs(loss)) * (tol + min(steps, 4000) * U) + 1e-37, "loss")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens, experts, k", [
    (1, 1, 1), (1, 64, 8), (2, 8, 2), (7, 3, 3), (33, 9, 4), (5, 16, 16), (130, 17, 5), (64, 60, 6), (65, 64, 1),
    (257, 100, 8), (40, 128, 32), (1000, 160, 6), (3, 256, 8), (77, 257, 2), (19, 511, 10), (300, 512, 8), (9, 1000, 3),
    (40, 1024, 32),
])
def test_route(cuda, dtype, tokens, experts, k):
    logits = (torch.randn((tokens, experts), generator=gen(tokens + experts)) * 2).to(dtype).to(cuda)
    for renormalize in (True, False):
        check_route(kl.moe_route(logits, k, renormalize=renormalize), logits, k, renormalize)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("experts", [8, 60, 64, 256, 300])
def test_route_masks_ties_and_odd_values(cuda, dtype, experts):
    """Closed experts, rows with nothing left, padding that holds NaN and infinities, equal logits, both
    zeros, the type's lowest value, NaN and infinities in a routed row."""
    tokens, k = 150, 4
    x = torch.randn((tokens, experts), generator=gen(experts)).to(dtype)
    x[torch.rand(x.shape, generator=gen(1)) < 0.4] = -math.inf
    x[3] = -math.inf
    x[4] = -math.inf
    x[4, experts - 1] = 0.5                      # fewer experts than k
    x[5] = 1.25                                  # all equal: the lowest indexes
    x[6] = 0.0
    x[6, 1::2] = -0.0                            # both zeros tie
    x[7] = torch.finfo(dtype).min                # the lowest finite value everywhere: a uniform row
    x[8] = torch.finfo(dtype).min
    x[8, 2] = 1.0
    x[9] = torch.finfo(dtype).max
    x[10] = math.nan
    x[11] = math.inf
    valid = torch.rand(tokens, generator=gen(2)) < 0.8
    valid[:10] = True
    valid[10:12] = False
    check_route(kl.moe_route(x.to(cuda), k, valid=valid.to(cuda)), x, k, True, valid)
    check_route(kl.moe_route(x.to(cuda), k, renormalize=False, valid=valid.to(cuda).to(torch.uint8)), x, k, False, valid)
    # NaN and +inf in a routed row reach its weights and the loss, and the ids stay in range.
    for bad in (math.nan, math.inf):
        y = torch.randn((3, experts), generator=gen(4)).to(dtype)
        y[1, 5] = bad
        r = kl.moe_route(y.to(cuda), k)
        ids, weights, _, _, _, _ = oracle.route(y, k)
        assert torch.equal(r.ids.cpu(), ids) and r.ids[1, 0] == 5
        assert r.weights[1].isnan().all() and r.weights[0::2].isfinite().all() and r.loss.isnan()


def test_route_nothing_routed(cuda):
    x = torch.full((5, 16), -math.inf, device=cuda)
    r = kl.moe_route(x, 2)
    assert (r.ids == -1).all() and (r.weights == 0).all() and (r.counts == 0).all() and r.tokens == 0 and r.loss == 0
    g = kl.moe_route_grad(x, r, torch.full((5, 2), math.nan, device=cuda), torch.tensor(math.nan, device=cuda))
    assert (g == 0).all()
    r = kl.moe_route(torch.empty((0, 16), device=cuda), 2)
    assert r.ids.shape == (0, 2) and (r.counts == 0).all() and r.tokens == 0 and r.loss == 0
    assert kl.moe_route_grad(torch.empty((0, 16), device=cuda), r).shape == (0, 16)


def test_route_strides_and_alignment(cuda):
    base = torch.randn((70, 80), generator=gen(6)).to(torch.bfloat16).to(cuda)
    for view in (base[:, 1:65], base[:, 8:72], base[::2, :64], base[3:4, 5:69]):
        check_route(kl.moe_route(view, 6), view, 6, True)
        r = kl.moe_route(view, 6)
        dw = torch.randn(r.weights.shape, generator=gen(7)).to(cuda)
        out = torch.full_like(base, 9.0)[:view.shape[0], 3:67]
        kl.moe_route_grad(view, r, dw, out=out)
        check_grad(out, view, 6, dw, None, True)


def check_grad(got, logits, k, dweights, dloss, renormalize, valid=None):
    want = oracle.route_grad(logits, k, dweights, dloss, renormalize, valid)
    _, w, counts, routed, _, probs = oracle.route(logits, k, renormalize, valid)
    tol = prob_tol(logits)
    experts = logits.shape[1]
    # Every product in the formula is off by its probabilities' relative error and a few roundings.
    size = torch.zeros_like(want)
    if dloss is not None and routed:
        a = abs(float(dloss)) * experts * counts.to(F64) / (k * routed * routed)
        size += probs * (a + (probs * a).sum(1, keepdim=True))
    if dweights is not None:
        ids = oracle.route(logits, k, renormalize, valid)[0]
        dw = torch.where(ids >= 0, dweights.cpu().to(F64), 0.0)
        total = (w * dw.abs()).sum(1, keepdim=True)
        size += probs * total
        size = size.scatter_add(1, ids.clamp(min=0).long(), w * (dw.abs() + total))
    close(got, want, want.abs() * HALF[logits.dtype] + size * (4 * tol + 16 * U) + 1e-37 +
          torch.finfo(logits.dtype).smallest_normal * HALF[logits.dtype] * 2, "dlogits")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens, experts, k", [(1, 1, 1), (1, 64, 8), (50, 8, 2), (33, 9, 4), (257, 100, 8), (700, 160, 6),
                                                (77, 257, 2), (21, 1000, 32)])
def test_route_grad(cuda, dtype, tokens, experts, k):
    logits = (torch.randn((tokens, experts), generator=gen(tokens)) * 1.5).to(dtype)
    logits[torch.rand(logits.shape, generator=gen(3)) < 0.2] = -math.inf
    valid = torch.rand(tokens, generator=gen(5)) < 0.9
    logits[~valid] = math.nan
    x = logits.to(cuda)
    dw = torch.randn((tokens, k), generator=gen(8)).to(cuda)
    dl = torch.tensor(3.0, device=cuda)
    for renormalize in (True, False):
        r = kl.moe_route(x, k, renormalize=renormalize, valid=valid.to(cuda))
        # What a closed slot's gradient holds is not read.
        dirty = torch.where(r.ids < 0, math.nan, dw)
        for a, b in ((dirty, dl), (None, dl), (dirty, None), (None, None)):
            got = kl.moe_route_grad(x, r, a, b, renormalize=renormalize, valid=valid.to(cuda))
            check_grad(got, logits, k, None if a is None else dw, None if b is None else 3.0, renormalize, valid)
    inplace = x.clone()
    want = kl.moe_route_grad(x, r, dirty, dl, renormalize=False, valid=valid.to(cuda))
    assert kl.moe_route_grad(inplace, r, dirty, dl, renormalize=False, valid=valid.to(cuda), out=inplace) is inplace
    assert torch.equal(inplace.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_grad_against_differences(cuda, renormalize):
    """Central differences of the float64 definition, the choice held by a gap between the logits."""
    tokens, experts, k, h = 3, 12, 3, 1e-5
    logits = torch.stack([torch.randperm(experts, generator=gen(i)).to(F64) * 0.3 for i in range(tokens)])
    dw, dl = torch.randn((tokens, k), generator=gen(9)).to(F64), 2.0
    x = logits.float().to(cuda)
    r = kl.moe_route(x, k, renormalize=renormalize)
    got = kl.moe_route_grad(x, r, dw.float().to(cuda), torch.tensor(dl, device=cuda), renormalize=renormalize)

    def value(z):
        _, w, _, _, loss, _ = oracle.route(z, k, renormalize)
        return (w * dw).sum().item() + dl * loss

    want = torch.zeros_like(logits)
    for t in range(tokens):
        for e in range(experts):
            up, down = x.cpu().to(F64), x.cpu().to(F64)
            up[t, e] += h
            down[t, e] -= h
            want[t, e] = (value(up) - value(down)) / (2 * h)
    # h^2 / 6 of a third derivative below 50, and the differences' own cancellation (2^-52 / h).
    close(got, want, 50 * h * h / 6 + 1e-9 + 1e-5 * want.abs() + 64 * U * dw.abs().max(), "against differences")


def test_route_many_tokens(cuda):
    """The two-kernel path at a size where every block takes several turns, against torch in float64 on the GPU."""
    tokens, experts, k = 20011, 96, 4
    x = torch.randn((tokens, experts), device=cuda, generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    r = kl.moe_route(x, k)
    order = torch.sort(x.double(), dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(r.ids, order.int())
    assert torch.equal(r.counts, torch.bincount(order.reshape(-1), minlength=experts).int())
    p = torch.softmax(x.double(), 1)
    loss = experts * (r.counts.double() / (k * tokens) * p.mean(0)).sum()
    assert abs(r.loss.item() - loss.item()) < 2e-5 * loss.item()
    again = kl.moe_route(x, k)
    assert all(torch.equal(a, b) for a, b in zip(r, again)), "results depend on timing"


# ------------------------------------------------------------------------------------ plan, dispatch, combine

@pytest.mark.parametrize("tokens, k, experts, block", [
    (1, 1, 1, 128), (1, 8, 64, 128), (37, 2, 16, 128), (300, 4, 8, 256), (129, 1, 3, 128), (2000, 3, 60, 128),
    (1500, 8, 256, 256), (700, 6, 1024, 128), (5000, 2, 2, 128),
])
def test_plan(cuda, tokens, k, experts, block):
    for fill in ("mixed", "one", "none"):
        ids = torch.randint(-1, experts, (tokens, k), generator=gen(tokens), dtype=torch.int32)
        if fill == "one":
            ids[:] = experts - 1
        elif fill == "none":
            ids[:] = -1
        ids[0, 0] = experts if fill == "mixed" else ids[0, 0]       # no such expert: dropped
        if fill == "mixed" and tokens > 1:
            ids[1, 0] = -(2 ** 31)
        plan = kl.moe_plan(ids.to(cuda), experts, block=block)
        rows, slots, groups = oracle.plan(ids, experts, block, kl.moe_rows(tokens * k, experts, block))
        assert torch.equal(plan.rows.cpu(), rows)
        assert torch.equal(plan.slots.cpu(), slots)
        assert torch.equal(plan.m_block_group.cpu(), groups)


def test_plan_of_nothing(cuda):
    plan = kl.moe_plan(torch.empty((0, 4), dtype=torch.int32, device=cuda), 8)
    assert plan.rows.shape == (0, 4) and plan.slots.numel() == 0 and plan.m_block_group.numel() == 0
    x = torch.empty((0, 64), device=cuda)
    assert kl.moe_dispatch(x, plan).shape == (0, 64)
    assert kl.moe_combine(torch.empty((0, 64), device=cuda), rows=plan.rows).shape == (0, 64)
    dy, dw = kl.moe_combine_grad(x, x, torch.empty((0, 4), device=cuda), rows=plan.rows, slots=plan.slots)
    assert dy.shape == (0, 64) and dw.shape == (0, 4)


def random_plan(cuda, tokens, k, experts, seed, block=128):
    ids = torch.randint(-1, experts, (tokens, k), generator=gen(seed), dtype=torch.int32).to(cuda)
    return kl.moe_plan(ids, experts, block=block)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8, torch.float8_e4m3fn])
@pytest.mark.parametrize("tokens, k, width", [(1, 1, 1), (5, 2, 7), (40, 3, 64), (33, 8, 1001), (129, 2, 2056)])
def test_dispatch(cuda, dtype, tokens, k, width):
    plan = random_plan(cuda, tokens, k, 6, tokens)
    x = torch.randint(0, 255, (tokens, (width + 3) * dtype.itemsize), generator=gen(1), dtype=torch.uint8).to(cuda).view(dtype)
    for view in (x[:, :width].contiguous(), x[:, 1:width + 1]):
        a = kl.moe_dispatch(view, plan)
        slots = plan.slots.long()
        want = view.contiguous().view(torch.uint8)[slots.clamp(min=0) // k]
        want = torch.where(slots[:, None] >= 0, want, 0)
        assert torch.equal(a.view(torch.uint8), want)
    out = torch.full((a.shape[0], width + 5), 1.0, device=cuda).to(dtype)
    guard = out.clone()
    kl.moe_dispatch(view, plan, out[:, 2:width + 2])
    assert torch.equal(out[:, 2:width + 2].contiguous().view(torch.uint8), want)
    for side in (slice(0, 2), slice(width + 2, None)):
        assert torch.equal(out[:, side].contiguous().view(torch.uint8), guard[:, side].contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens, k, width", [(1, 1, 1), (1, 8, 256), (5, 2, 7), (40, 3, 64), (33, 9, 1001), (70, 32, 96),
                                              (17, 4, 4104)])
def test_combine_and_gradient(cuda, dtype, tokens, k, width):
    plan = random_plan(cuda, tokens, k, 5, tokens + k)
    y = torch.randn((plan.slots.numel(), width), generator=gen(2)).to(dtype)
    y[plan.slots.cpu() < 0] = math.nan            # padding rows are nobody's
    w = torch.randn((tokens, k), generator=gen(3))
    dout = torch.randn((tokens, width), generator=gen(4)).to(dtype)
    rows = plan.rows.cpu().long()
    live = (rows >= 0)[..., None]
    picked = torch.where(live, y[rows.clamp(min=0)].to(F64), 0.0)
    yd, wd = y.to(cuda), w.to(cuda)
    for weights in (wd, None):
        w64 = w.to(F64) if weights is not None else torch.ones_like(w, dtype=F64)
        want = (w64[..., None] * picked).sum(1)
        size = (w64[..., None] * picked).abs().sum(1)
        got = kl.moe_combine(yd, weights, rows=plan.rows)
        # k products and sums in fp32, one rounding to the type (or its smallest step).
        close(got, want, size * (k + 1) * U + want.abs() * HALF[dtype] * (1 + 2 * k * U) + torch.finfo(dtype).smallest_normal * HALF[dtype] * 2,
              "combine")
        dy, dw = kl.moe_combine_grad(dout.to(cuda), yd, weights, rows=plan.rows, slots=plan.slots)
        slots = plan.slots.cpu().long()
        at = slots.clamp(min=0)
        want = torch.where(slots[:, None] >= 0, w64.reshape(-1)[at][:, None] * dout.to(F64)[at // k], 0.0)
        close(dy, want, want.abs() * (HALF[dtype] + 2 * U) + torch.finfo(dtype).smallest_normal * HALF[dtype] * 2, "dy")
        if weights is None:
            assert dw is None
            continue
        terms = dout.to(F64)[:, None, :] * picked
        # A thread's own terms one after another, then 5 shuffles and 8 warps.
        close(dw, terms.sum(2), terms.abs().sum(2) * (width / 256 * 8 + 32) * U + 1e-37, "dweights")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_combine_in_slot_order(cuda, dtype):
    y = torch.randn((6, 3, 40), generator=gen(1)).to(dtype).to(cuda)
    w = torch.rand((6, 3), generator=gen(2)).to(cuda)
    dout = torch.randn((6, 40), generator=gen(3)).to(dtype).to(cuda)
    want = (w.double()[..., None] * y.double()).sum(1).cpu()
    close(kl.moe_combine(y, w), want, (w.double()[..., None] * y.double()).abs().sum(1).cpu() * 4 * U + want.abs() * HALF[dtype] * 1.001, "out")
    dy, dw = kl.moe_combine_grad(dout, y, w)
    assert dy.shape == y.shape
    want = (w.double()[..., None] * dout.double()[:, None]).cpu()
    close(dy, want, want.abs() * (HALF[dtype] + 2 * U), "dy")
    close(dw, (dout.double()[:, None] * y.double()).sum(2).cpu(), (dout.double()[:, None] * y.double()).abs().sum(2).cpu() * 48 * U, "dw")


def test_combine_strides_and_repeated_rows(cuda):
    base = torch.randn((200, 90), generator=gen(1)).to(torch.bfloat16).to(cuda)
    rows = torch.randint(-1, 100, (12, 4), generator=gen(2), dtype=torch.int32).to(cuda)
    rows[3] = 7                                   # one row for every slot of a token
    rows[4, 1] = 100                              # behind the last row: adds nothing
    w = torch.rand((12, 4), generator=gen(3)).to(cuda)
    for y in (base[::2, 8:72], base[:100, 1:65], base[:100, 3:90]):
        out = torch.full((12, 99), 5.0, device=cuda, dtype=torch.bfloat16)
        kl.moe_combine(y, w, rows=rows, out=out[:, 1:1 + y.shape[1]])
        live = ((rows >= 0) & (rows < 100))[..., None]
        picked = torch.where(live, y[rows.clamp(0, 99).long()].double(), 0.0)
        terms = w.double()[..., None] * picked
        close(out[:, 1:1 + y.shape[1]], terms.sum(1).cpu(), terms.abs().sum(1).cpu() * 5 * U + terms.sum(1).abs().cpu() * HALF[y.dtype] * 1.001)
        assert (out[:, 0] == 5).all() and (out[:, 1 + y.shape[1]:] == 5).all()


# ------------------------------------------------------------------------------------ 4-bit weights

def int4_case(cuda, n, k, group, dtype, zeros, experts=0, seed=0, scale_dtype=None):
    lead = (experts,) if experts else ()
    q = torch.randint(0, 256, (*lead, n, k // 2), generator=gen(seed), dtype=torch.uint8)
    s = (torch.rand((*lead, n, -(-k // group)), generator=gen(seed + 1)) * 0.02 + 0.001).to(scale_dtype or dtype)
    z = torch.randint(0, 128 if zeros == "wide" else 16, s.shape, generator=gen(seed + 2), dtype=torch.uint8) if zeros else None
    return q.to(cuda), s.to(cuda), None if z is None else z.to(cuda)


def gemv_tol(x, w, want, k, dtype):
    """x enters as fixed-point numbers, off by at most 2^-22 of its group's largest. A group's products are
    summed exactly; each group's sum takes 3 roundings to scale and 3 to join its three digits, then at
    most k / 32 sums, 16 warps and 8 blocks are added in fp32; one rounding to the type. With three tokens
    and more, x and q - z enter as they are; a group of up to 128 is 8 steps of 16 products, each step's sum cut off
    below 2 U of what the group's products sum to, so 16 U a group, one rounding to scale it, and the same sums after."""
    x = x.to(F64).abs()
    if x.shape[0] == 0:
        return torch.zeros_like(want)
    fixed = 2.0 ** -22 * x.max(-1, keepdim=True)[0] * w.abs().sum(1)
    size = x @ w.abs().T
    return fixed + (size + fixed) * (k / 32 + 32) * U + want.abs() * HALF[dtype] * 1.001 + torch.finfo(dtype).smallest_normal * HALF[dtype] * 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128, 384])
@pytest.mark.parametrize("tokens, n, k", [(1, 1, 32), (1, 16, 128), (2, 17, 96), (3, 100, 1056), (8, 64, 4128), (9, 33, 512),
                                          (16, 130, 2048), (17, 40, 160), (33, 50, 256), (70, 20, 1024)])
def test_gemv_int4(cuda, dtype, group, tokens, n, k):
    for zeros in (None, "narrow", "wide"):
        q, s, z = int4_case(cuda, n, k, group, dtype, zeros, seed=tokens + n)
        x = torch.randn((tokens, k), generator=gen(k)).to(dtype)
        w = oracle.int4_weights(q, s, z, group)
        want = x.to(F64) @ w.T
        close(kl.gemv_int4(x.to(cuda), q, s, z, group=group), want, gemv_tol(x, w, want, k, dtype), f"zeros {zeros}")
    got = kl.gemv_int4(x.to(cuda), q, s.float(), z, group=group, out_dtype=torch.float32)
    close(got, want, gemv_tol(x, w, want, k, torch.float32), "fp32 scales and out")


@pytest.mark.parametrize("tokens, n, k, group", [
    (1, 16 * 148 * 14 + 5, 2048, 128),    # every block has several tiles, cut between the warps
    (2, 16 * 148 * 21, 512, 32),          # a full batch of 16 tiles and a rest, one unit a tile
    (1, 16 * 148 * 3, 1536, 64), (5, 16 * 300 + 1, 2560, 64), (13, 10007, 4128, 64), (16, 16 * 700, 8192, 128),
    (33, 16 * 200, 1056, 32), (3, 40, 16384, 128), (16, 64, 32768, 32), (1, 32, 65536, 64), (2, 8192, 8192, 256),
    (5, 40, 65536, 64), (12, 24, 40960, 128), (3, 16 * 148, 36896, 32),    # x of 8 or 16 tokens does not fit
])
def test_gemv_int4_many_tiles(cuda, tokens, n, k, group):
    """Sizes at which blocks have several tiles, tiles are shared between warps, K is split over a cluster."""
    g = torch.Generator("cuda").manual_seed(n + k)
    q = torch.randint(0, 256, (n, k // 2), generator=g, device=cuda, dtype=torch.uint8)
    s = (torch.rand((n, -(-k // group)), generator=g, device=cuda) * 0.02 + 0.001).bfloat16()
    z = torch.randint(0, 16, s.shape, generator=g, device=cuda, dtype=torch.uint8)
    x = torch.randn((tokens, k), generator=g, device=cuda).bfloat16()
    codes = torch.stack([q & 15, q >> 4], -1).flatten(-2).double()
    at = torch.arange(k, device=cuda) // group
    w = (codes - z.double()[:, at]) * s.double()[:, at]
    want = x.double() @ w.T
    tol = gemv_tol(x, w, want, k, torch.bfloat16)
    for _ in range(2):
        close(kl.gemv_int4(x, q, s, z, group=group), want.cpu(), tol.cpu())


def test_gemv_int4_by_expert_many_tiles(cuda):
    """Blocks whose tiles belong to several experts, experts with several passes of tokens."""
    g = torch.Generator("cuda").manual_seed(5)
    for tokens, k, experts, n, width, group in ((1, 8, 64, 4096, 2048, 128), (16, 4, 64, 2064, 1536, 32), (40, 2, 3, 1000, 768, 64),
                                                (300, 2, 5, 500, 512, 128)):
        q = torch.randint(0, 256, (experts, n, width // 2), generator=g, device=cuda, dtype=torch.uint8)
        s = (torch.rand((experts, n, -(-width // group)), generator=g, device=cuda) * 0.02 + 0.001).half()
        ids = torch.randint(-1, experts, (tokens, k), generator=g, device=cuda, dtype=torch.int32)
        x = torch.randn((tokens, k, width), generator=g, device=cuda).half()
        got = kl.gemv_int4(x, q, s, group=group, ids=ids)
        at = torch.arange(width, device=cuda) // group
        assert (got[ids < 0] == 0).all()
        for e in range(experts):
            mine = ids == e
            codes = torch.stack([q[e] & 15, q[e] >> 4], -1).flatten(-2).double()
            w = (codes - 8) * s[e].double()[:, at]
            want = x[mine].double() @ w.T
            close(got[mine], want.cpu(), gemv_tol(x[mine], w, want, width, torch.float16).cpu(), f"expert {e}")


def test_gemv_int4_every_code(cuda):
    """One-hot rows of x read every weight alone: exact results, so a wrong nibble order shows."""
    n, k = 24, 256
    for dtype in (torch.bfloat16, torch.float16):
        for group in (32, 64, 128):
            q, _, z = int4_case(cuda, n, k, group, dtype, "narrow", seed=group)
            s = torch.ones((n, k // group), dtype=dtype, device=cuda)
            got = kl.gemv_int4(torch.eye(k, dtype=dtype, device=cuda), q, s, z, group=group)
            assert torch.equal(got.cpu().to(F64), oracle.int4_weights(q, s, z, group).T)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 2, 5, 16])
def test_gemv_int4_any_zero_point(cuda, dtype, tokens):
    """Zero points up to 255, which 8 bits of a bf16 cannot hold beside a code."""
    n, k, group = 50, 640, 64
    q, s, _ = int4_case(cuda, n, k, group, dtype, None, seed=tokens)
    z = torch.randint(0, 256, s.shape, generator=gen(tokens), dtype=torch.uint8)
    z[:, 0], z[:16], z[3, 1] = 127, z[:16] % 128, 128
    x = torch.randn((tokens, k), generator=gen(9)).to(dtype)
    w = oracle.int4_weights(q, s, z, group)
    want = x.to(F64) @ w.T
    close(kl.gemv_int4(x.to(cuda), q, s, z.to(cuda), group=group), want, gemv_tol(x, w, want, k, dtype))
    # Codes and zero points alone: every weight exactly.
    eye = torch.eye(k, dtype=dtype, device=cuda)[:tokens]
    got = kl.gemv_int4(eye, q, torch.ones_like(s), z.to(cuda), group=group, out_dtype=torch.float32)
    assert torch.equal(got.cpu().to(F64), oracle.int4_weights(q, torch.ones_like(s), z, group).T[:tokens])


def test_gemv_int4_strides(cuda):
    n, k = 48, 512
    q, s, z = int4_case(cuda, 2 * n, 2 * k, 64, torch.bfloat16, "narrow", seed=3)
    base = torch.randn((12, 2 * k), generator=gen(1)).to(torch.bfloat16).to(cuda)
    x = base[::2, 8:8 + k]
    qv, sv, zv = q[::2, 32:32 + k // 2], s[::2, 1:9], z[::2, 3:11]
    out = torch.full((6, n + 3), 4.0, dtype=torch.bfloat16, device=cuda)
    kl.gemv_int4(x, qv, sv, zv, group=64, out=out[:, 1:n + 1])
    w = oracle.int4_weights(qv, sv, zv, 64)
    want = x.cpu().to(F64) @ w.T
    close(out[:, 1:n + 1], want, gemv_tol(x.cpu(), w, want, k, torch.bfloat16))
    assert (out[:, 0] == 4).all() and (out[:, n + 1:] == 4).all()
    with pytest.raises(kl.KlError):
        kl.gemv_int4(base[:, 4:4 + k], qv, sv, zv, group=64)   # 8-byte aligned rows


def test_gemv_int4_infinities_stay_in_their_row(cuda):
    q, s, _ = int4_case(cuda, 40, 256, 128, torch.bfloat16, None)
    x = torch.randn((9, 256), generator=gen(1)).to(torch.bfloat16)
    clean = kl.gemv_int4(x.to(cuda), q, s)
    x[2, 5], x[8, 100] = math.inf, math.nan
    got = kl.gemv_int4(x.to(cuda), q, s)
    rest = [0, 1, 3, 4, 5, 6, 7]
    assert torch.equal(got[rest], clean[rest]) and not got[2].isfinite().any() and got[8].isnan().all()


def test_gemv_int4_nothing(cuda):
    q, s, _ = int4_case(cuda, 8, 64, 32, torch.bfloat16, None)
    assert kl.gemv_int4(torch.empty((0, 64), dtype=torch.bfloat16, device=cuda), q, s, group=32).shape == (0, 8)
    none = kl.gemv_int4(torch.empty((3, 0), dtype=torch.bfloat16, device=cuda), q[:, :0], s[:, :0], group=32)
    assert none.shape == (3, 8) and (none == 0).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens, k, experts, n, width", [
    (1, 1, 1, 16, 64), (1, 8, 64, 40, 256), (4, 2, 8, 33, 1024), (16, 4, 6, 20, 160), (60, 3, 5, 17, 128), (1, 4, 2, 30, 512),
])
def test_gemv_int4_by_expert(cuda, group, tokens, k, experts, n, width):
    for dtype, zeros in ((torch.bfloat16, None), (torch.float16, "narrow")):
        q, s, z = int4_case(cuda, n, width, group, dtype, zeros, experts, seed=tokens)
        # Any ids: repeated, none, out of range.
        ids = torch.randint(-1, experts + 1, (tokens, k), generator=gen(tokens + k), dtype=torch.int32)
        w = oracle.int4_weights(q, s, z, group)
        live = (ids >= 0) & (ids < experts)
        for shape in ((tokens, width), (tokens, k, width)):
            x = torch.randn(shape, generator=gen(5)).to(dtype)
            got = kl.gemv_int4(x.to(cuda), q, s, z, group=group, ids=ids.to(cuda))
            assert got.shape == (tokens, k, n)
            for t in range(tokens):
                for j in range(k):
                    if not live[t, j]:
                        assert (got[t, j] == 0).all()
                        continue
                    row = (x[t, j] if x.dim() == 3 else x[t])[None]
                    m = w[ids[t, j]]
                    want = row.to(F64) @ m.T
                    close(got[t, j][None], want, gemv_tol(row, m, want, width, dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("width", [2, 7, 1023, 2046, 4095, 4100, 4104])
@pytest.mark.parametrize("shift", [0, 1])
def test_rows_of_any_alignment(cuda, dtype, width, shift):
    """Rows that begin anywhere, in pitches that fit no vector: copies exactly, sums against 64 bits, nothing beside
    the rows written."""
    tokens, experts, k = 37, 5, 2
    ids = torch.randint(-1, experts, (tokens, k), generator=gen(width), dtype=torch.int32).to(cuda)
    plan = kl.moe_plan(ids, experts)
    m = plan.slots.shape[0]
    x = torch.randn((tokens, width + 3), generator=gen(1)).to(dtype).to(cuda)[:, shift:shift + width]
    room = torch.full((m, width + 5), 9.0, dtype=dtype, device=cuda)
    y = kl.moe_dispatch(x, plan, out=room[:, shift:shift + width])
    slots = plan.slots.long()
    want = torch.where((slots >= 0)[:, None], x[slots.clamp(min=0) // k], 0)
    assert torch.equal(y, want) and (room[:, :shift] == 9).all() and (room[:, shift + width:] == 9).all()
    weights = torch.rand((tokens, k), generator=gen(2)).to(cuda)
    live = (plan.rows >= 0).double() * weights.double()
    rows = plan.rows.long().clamp(min=0)
    out = kl.moe_combine(y, weights, rows=plan.rows)
    want = (live[..., None] * y.double()[rows]).sum(1)
    close(out, want.cpu(), (want.abs() * HALF[dtype] * 1.001 + 3 * U * (live[..., None] * y.double()[rows].abs()).sum(1) + 2.0 ** -25).cpu())
    dy, dw = kl.moe_combine_grad(x, y, weights, rows=plan.rows, slots=plan.slots)
    wanted = x.double()[slots.clamp(min=0) // k] * weights.double().flatten()[slots.clamp(min=0)][:, None] * (slots >= 0)[:, None]
    close(dy, wanted.cpu(), (wanted.abs() * (HALF[dtype] * 1.001 + U) + 2.0 ** -25).cpu())
    products = x.double()[:, None] * y.double()[rows] * (plan.rows >= 0)[..., None]
    # A thread's products one after another, then 8 exchanges: at most width / 256 + 16 + 16 roundings.
    close(dw, products.sum(-1).cpu(), (products.abs().sum(-1) * (width / 256 + 32) * U).cpu())


# ------------------------------------------------------------------------------------ streams, graphs, together

FIRST_IN_CAPTURE = """
import torch
import maia_b200 as kl
d = torch.device("cuda", 0)
x = torch.randn((100, 64), device=d)
q = torch.randint(0, 256, (4096, 1024), device=d, dtype=torch.uint8)
s, v = torch.rand((4096, 16), device=d).bfloat16(), torch.randn((3, 2048), device=d).bfloat16()
torch.cuda.synchronize()
def step():
    r = kl.moe_route(x, 4, renormalize=True)
    plan = kl.moe_plan(r.ids, 64)
    return kl.moe_combine(kl.moe_dispatch(x, plan), r.weights, rows=plan.rows), kl.gemv_int4(v, q, s)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
"""


def test_first_call_may_be_captured(cuda):
    """A process whose first call of each operator is made while a graph is captured."""
    done = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE], cwd=pathlib.Path(__file__).parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_graph_replay_and_streams(cuda):
    """The whole path captured on a side stream and replayed with new inputs in place: the results
    are the eager call's, bit for bit."""
    tokens, experts, k, width, n = 50, 8, 2, 256, 192
    q, s, z = int4_case(cuda, n, width, 64, torch.bfloat16, "narrow", experts)
    logits = torch.empty((tokens, experts), device=cuda)
    x = torch.empty((tokens, width), dtype=torch.bfloat16, device=cuda)

    def step():
        r = kl.moe_route(logits, k)
        plan = kl.moe_plan(r.ids, experts)
        a = kl.moe_dispatch(x, plan)
        y = kl.gemv_int4(x, q, s, z, group=64, ids=r.ids)
        out = kl.moe_combine(y, r.weights)
        dy, dw = kl.moe_combine_grad(out, y, r.weights)
        g = kl.moe_route_grad(logits, r, dw, r.loss)
        back = kl.moe_combine(a, rows=plan.rows)
        return (*r, *plan, a, y, out, dy, dw, g, back)

    def fill(seed):
        logits.copy_(torch.randn(logits.shape, generator=gen(seed)))
        x.copy_(torch.randn(x.shape, generator=gen(seed + 1)))

    fill(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, twin = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.cuda.graph(twin):
        outs2 = step()
    for seed in (11, 12, 13):
        fill(seed)
        torch.cuda.synchronize()
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        other = torch.cuda.Stream()
        with torch.cuda.stream(other):
            twin.replay()                          # both graphs at once: nothing is shared
        torch.cuda.synchronize()
        for a, b, c in zip(outs, outs2, step()):
            assert torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))
            assert torch.equal(a.reshape(-1).view(torch.uint8), c.reshape(-1).view(torch.uint8))


def test_stream_argument(cuda):
    """A raw stream handle that is not torch's current stream: the call is ordered on it."""
    x = torch.randn((3000, 64), generator=gen(1)).to(cuda)
    want = kl.moe_route(x, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        got = kl.moe_route(x, 4, stream=side.cuda_stream)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_routed_experts_with_grouped_gemm(cuda):
    """Prefill: route, plan, dispatch, gemm_grouped, combine against the experts applied one token at a time."""
    tokens, experts, k, width, n = 200, 6, 2, 256, 320
    x = torch.randn((tokens, width), generator=gen(1)).to(torch.bfloat16).to(cuda)
    w = (torch.randn((experts, n, width), generator=gen(2)) / 16).to(torch.bfloat16).to(cuda)
    logits = torch.randn((tokens, experts), generator=gen(3)).to(cuda)
    for block, algo in ((128, kl.ALGO_1CTA), (256, kl.ALGO_2CTA)):
        r = kl.moe_route(logits, k)
        plan = kl.moe_plan(r.ids, experts, block=block)
        a = kl.moe_dispatch(x, plan)
        y = kl.gemm_grouped(a, w, plan.m_block_group, out_dtype=torch.float32, algo=algo)
        out = kl.moe_combine(y, r.weights, rows=plan.rows)
        torch.cuda.synchronize()
        assert kl.read_status() == 0
        products = torch.einsum("tw,tjnw->tjn", x.double(), w.double()[r.ids.long()])
        want = (r.weights.double()[..., None] * products).sum(1).cpu()
        size = (r.weights.double()[..., None] * torch.einsum("tw,tjnw->tjn", x.double().abs(), w.double().abs()[r.ids.long()])).sum(1).cpu()
        close(out, want, size * (width / 16 + 8) * 2.0 ** -22, f"block {block}")


def test_routed_experts_with_4_bit_weights(cuda):
    """Decode: route, two products of each token's experts with an activation between, combine."""
    tokens, experts, k, width, hidden = 5, 8, 2, 256, 384
    up = int4_case(cuda, hidden, width, 128, torch.bfloat16, None, experts, seed=1)
    down = int4_case(cuda, width, hidden, 128, torch.bfloat16, "narrow", experts, seed=2)
    x = torch.randn((tokens, width), generator=gen(1)).to(torch.bfloat16).to(cuda)
    r = kl.moe_route(torch.randn((tokens, experts), generator=gen(2)).to(cuda), k)
    h = torch.nn.functional.silu(kl.gemv_int4(x, *up, ids=r.ids))
    y = kl.gemv_int4(h, *down, ids=r.ids)
    out = kl.moe_combine(y, r.weights)
    wu, wd = oracle.int4_weights(*up, 128), oracle.int4_weights(*down, 128)
    ids = r.ids.cpu().long()
    want_h = torch.einsum("tw,tjnw->tjn", x.cpu().to(F64), wu[ids])
    close(h, torch.nn.functional.silu(want_h), want_h.abs() * 3 * HALF[torch.bfloat16] + 1e-2, "h")
    want_y = torch.einsum("tjw,tjnw->tjn", h.cpu().to(F64), wd[ids])
    size = torch.einsum("tjw,tjnw->tjn", h.cpu().to(F64).abs(), wd[ids].abs())
    fixed = 2.0 ** -22 * h.cpu().to(F64).abs().max() * wd.abs().sum(2).max()
    close(y, want_y, fixed + size * 64 * U + want_y.abs() * HALF[torch.bfloat16] * 1.001, "y")
    terms = r.weights.cpu().to(F64)[..., None] * y.cpu().to(F64)
    close(out, terms.sum(1), terms.abs().sum(1) * 4 * U + terms.sum(1).abs() * HALF[torch.bfloat16] * 1.001, "out")


# ------------------------------------------------------------------------------------ torch.ops.kl with gradients

@pytest.mark.parametrize("renormalize", [True, False])
def test_layer_gradients_through_torch_ops(cuda, renormalize):
    """A training step through torch.ops.kl: route, plan, dispatch, the experts (torch), combine and the balance
    loss; every gradient against torch's autograd over the same layer in float64, the choice held fixed."""
    import maia_b200.torch_ops  # noqa: F401

    tokens, experts, k, width, n = 70, 6, 2, 48, 40
    logits = torch.randn((tokens, experts), generator=gen(1)).to(cuda).requires_grad_()
    x = torch.randn((tokens, width), generator=gen(2)).to(cuda).requires_grad_()
    w = (torch.randn((experts, n, width), generator=gen(3)) / 7).to(cuda).requires_grad_()
    head = torch.randn((tokens, n), generator=gen(4)).to(cuda)
    ids, weights, counts, routed, loss = torch.ops.kl.moe_route(logits, k, renormalize)
    assert not ids.requires_grad and not counts.requires_grad and loss.requires_grad
    rows, slots, groups = torch.ops.kl.moe_plan(ids, experts)
    a = torch.ops.kl.moe_dispatch(x, rows, slots)
    y = torch.cat([a[128 * i:128 * i + 128] @ (w[g].T if g >= 0 else 0 * w[0].T) for i, g in enumerate(groups.tolist())])
    out = torch.ops.kl.moe_combine(y, weights, rows, slots)
    ((out * head).sum() + 0.3 * loss).backward()

    l64, x64, w64 = (t.detach().double().requires_grad_() for t in (logits, x, w))
    p = torch.softmax(l64, 1)
    sel = p.gather(1, ids.long())
    if renormalize:
        sel = sel / sel.sum(1, keepdim=True)
    out64 = (sel[..., None] * torch.einsum("tw,tjnw->tjn", x64, w64[ids.long()])).sum(1)
    loss64 = experts * (counts.double() / (k * tokens) * p.mean(0)).sum()
    ((out64 * head.double()).sum() + 0.3 * loss64).backward()
    # fp32 throughout, torch's own products among it: sums of up to tokens * k * width terms of size 1.
    for name, mine, theirs in (("logits", logits, l64), ("x", x, x64), ("w", w, w64)):
        close(mine.grad, theirs.grad.cpu(), 256 * U * theirs.grad.abs().max().item() * 8, name)
    close(loss, loss64.detach().cpu(), 1e-5, "loss")


def test_gradients_that_only_one_output_uses(cuda):
    import maia_b200.torch_ops  # noqa: F401

    logits = torch.randn((40, 8), generator=gen(1)).to(cuda).requires_grad_()
    _, weights, _, _, loss = torch.ops.kl.moe_route(logits, 2)
    (g,) = torch.autograd.grad(loss, logits, retain_graph=True)
    check_grad(g, logits.detach(), 2, None, 1.0, True)
    dw = torch.randn((40, 2), generator=gen(2)).to(cuda)
    (g,) = torch.autograd.grad(weights, logits, dw)
    check_grad(g, logits.detach(), 2, dw, None, True)
    # Rows without slots: the sum runs, its gradient is refused.
    rows = torch.arange(8, dtype=torch.int32, device=cuda).view(4, 2)
    y = torch.randn((8, 16), device=cuda, requires_grad=True)
    out = torch.ops.kl.moe_combine(y, None, rows)
    with pytest.raises(RuntimeError, match="slots"):
        out.sum().backward()
    # Slot order, no weights: a broadcast gradient.
    y = torch.randn((4, 2, 16), device=cuda, requires_grad=True)
    torch.ops.kl.moe_combine(y).sum().backward()
    assert (y.grad == 1).all()
    q, s, _ = int4_case(cuda, 16, 64, 32, torch.bfloat16, None)
    x = torch.randn((2, 64), generator=gen(3)).bfloat16().to(cuda)
    assert torch.equal(torch.ops.kl.gemv_int4(x, q, s, None, 32), kl.gemv_int4(x, q, s, group=32))


def test_training_step_in_a_graph(cuda):
    """Forward and backward through torch.ops.kl, captured and replayed on new values: the eager step's bits."""
    import maia_b200.torch_ops  # noqa: F401

    tokens, experts, k, width = 70, 16, 3, 136
    logits = torch.empty((tokens, experts), device=cuda, requires_grad=True)
    x = torch.empty((tokens, width), device=cuda, dtype=torch.bfloat16, requires_grad=True)

    def fill(seed):
        with torch.no_grad():
            logits.copy_(torch.randn(logits.shape, generator=gen(seed)))
            x.copy_(torch.randn(x.shape, generator=gen(seed + 1)))

    def step():
        ids, weights, _, _, loss = torch.ops.kl.moe_route(logits, k)
        rows, slots, _ = torch.ops.kl.moe_plan(ids, experts)
        y = torch.ops.kl.moe_dispatch(x, rows, slots)
        out = torch.ops.kl.moe_combine(y, weights, rows, slots)
        return torch.autograd.grad(out.float().square().sum() + loss, [logits, x])

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for seed in (3, 9):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
