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
