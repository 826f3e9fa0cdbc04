"""The projection with adapters: what z = scaling_i x_t A_i^T keeps, whatever the number of tokens.

z is a sum in fp32 and enters the product with B as fp32 holds it, in fp32's range, in both types.
"""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16 = torch.bfloat16, torch.float16
TOKENS = [1, 16, 40, 128, 129, 300, 1100, 2500]


@pytest.mark.parametrize("outer", [16, 264, 4104])
@pytest.mark.parametrize("power", [-16, -12, 0, 8, 20, 28])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens", TOKENS)
def test_z_has_the_bits_and_the_range_of_fp32(tokens, dtype, power, outer):
    """z_0 = h + m + l, z_1 = h, z_2 = m with l = 2^-9 m = 1.5 2^-18 h, times 2^power; y = (z_0 - z_1 - z_2) 2^-power.

    Every partial sum, in any order, is a multiple of 2^-19 h below 2 h: exact in fp32.  Of z_0 l is what
    two bf16 terms leave, and 2^power takes z out of fp16's range or its normal numbers.
    """
    inner, rank, adapters = 24, 24, 3
    size = torch.exp2(torch.arange(tokens, device=DEV) % 3 - 1.0)  # of h
    x = torch.zeros(tokens, inner, device=DEV)
    for column, part in ((1, 1.0), (9, 1.5 * 2.0 ** -9), (18, 1.5 * 2.0 ** -18)):
        x[:, column] = size * part
    a_power = max(-14, min(14, power))
    scaling = torch.tensor([1.0, 2.0 ** (power - a_power), 1.0], device=DEV)
    a = torch.zeros(adapters, rank, inner, device=DEV)
    for r, columns in ((0, [1, 9, 18]), (7, [1]), (19, [9])):
        a[1, r, columns] = 2.0 ** a_power
    b_power = max(-14, min(14, -power))
    b = torch.zeros(adapters, outer, rank, device=DEV)
    b[1, :, 0] = 2.0 ** b_power
    b[1, :, [7, 19]] = -2.0 ** b_power
    b[1, ::2] *= -1.0
    x, a, b = x.to(dtype), a.to(dtype), b.to(dtype)
    w = torch.zeros(outer, inner, dtype=dtype, device=DEV)
    ids = torch.ones(tokens, dtype=torch.int32, device=DEV)
    ids[3::5] = 2  # (zeros)
    want = torch.where(ids == 1, size * 1.5 * 2.0 ** (power + b_power - 18), 0.0)
    want = want.unsqueeze(1).expand(tokens, outer).clone()
    want[:, ::2] *= -1.0
    y = ops.adapted_linear(x, w, a, b, ids, scaling=scaling)
    assert torch.equal(y.float(), want.to(dtype).float())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("inner,outer,adapters,rank", [(512, 256, 3, 16), (264, 4104, 5, 40),
                                                       (1032, 520, 2, 128)])
@pytest.mark.parametrize("tokens", TOKENS)
def test_adapters_alone(tokens, inner, outer, adapters, rank, dtype):
    """W = 0, weights of wide range.  Each addition is off by at most a unit in the last place, the scaling's product
    by half a unit; B in fp16 may be two terms, whose dropped product is below 2^-26 of z B:
      |dz| <= (K + 1) 2^-23 s |x| |A|^T,  |dy| <= 80 ceil(rank / 16) 2^-23 |z| |B|^T + |dz| |B|^T + u |y|
    (five products of 16 columns for 16 ranks), and half the type's smallest value."""
    g = torch.Generator(device=DEV).manual_seed(tokens + rank)

    def normal(*shape, spread=0):
        v = torch.randn(*shape, generator=g, device=DEV) * shape[-1] ** -0.5
        return (v * torch.exp2(torch.randint(-spread, spread + 1, shape, generator=g, device=DEV)
                               .float())).to(dtype)

    x, a, b = normal(tokens, inner), normal(adapters, rank, inner), normal(adapters, outer, rank, spread=6)
    s = torch.exp2(torch.randint(-8, 9, (adapters,), generator=g, device=DEV).float()) * 1.37
    ids = torch.randint(-1, adapters, (tokens,), generator=g, device=DEV)
    w = torch.zeros(outer, inner, dtype=dtype, device=DEV)
    y = ops.adapted_linear(x, w, a, b, ids, scaling=s)
    u, t = torch.finfo(dtype).eps / 2, 2.0 ** -23
    tiny = torch.finfo(dtype).smallest_normal * u
    for i in range(-1, adapters):
        mine = ids == i
        if i < 0:
            assert not bool(y[mine].any())
            continue
        xi, ai, bi, si = x[mine].double(), a[i].double(), b[i].double(), float(s[i])
        z = si * (xi @ ai.t())
        dz = (inner + 1) * t * si * (xi.abs() @ ai.abs().t())
        want = z @ bi.t()
        bound = 80 * ((rank + 15) // 16) * t * (z.abs() @ bi.abs().t()) + dz @ bi.abs().t()
        bound = (bound + u * want.abs() + tiny) * (1 + u)
        off = (y[mine].double() - want).abs()
        assert bool((off <= bound).all()), f"off by {(off / bound).max().item():.3g} bounds"


@pytest.mark.parametrize("tokens", [128, 129, 1100])
def test_one_token_far_above_the_others(tokens):
    """fp16: a z of 7e4 against B of 1e-3 is 70 in any batch."""
    x = torch.zeros(tokens, 16, dtype=F16, device=DEV)
    x[:, 0] = 1.0
    x[tokens // 2, 0] = 700.0
    a = torch.zeros(1, 8, 16, dtype=F16, device=DEV)
    a[0, 0, 0] = 100.0
    b = torch.zeros(1, 40, 8, dtype=F16, device=DEV)
    b[0, ::2, 0] = 2.0 ** -10  # (zero elsewhere: an infinity times it would be a NaN)
    w = torch.zeros(40, 16, dtype=F16, device=DEV)
    y = ops.adapted_linear(x, w, a, b, torch.zeros(tokens, dtype=torch.int32, device=DEV))
    want = torch.zeros(tokens, 40, device=DEV)
    want[:, ::2] = (x[:, :1].float() * 100.0) * 2.0 ** -10
    assert torch.equal(y, want.to(F16))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 128])
@pytest.mark.parametrize("tokens", TOKENS)
def test_infinite_factor(tokens, rank, dtype):
    """x, A and B above 0 and an infinite factor of one adapter: its tokens are infinite, none is a NaN."""
    x = torch.full((tokens, 24), 0.5, dtype=dtype, device=DEV)
    a = torch.full((2, rank, 24), 0.25, dtype=dtype, device=DEV)
    b = torch.full((2, 136, rank), 1.5, dtype=dtype, device=DEV)
    w = torch.ones(136, 24, dtype=dtype, device=DEV)
    ids = (torch.arange(tokens, device=DEV) % 3 - 1).int()
    y = ops.adapted_linear(x, w, a, b, ids,
                           scaling=torch.tensor([float("inf"), 2.0], device=DEV)).float()
    assert bool((y[ids == 0] == float("inf")).all())
    assert bool((y[ids == -1] == 12.0).all())
    want = torch.tensor(12.0 + 9.0 * rank).to(dtype).item()  # (a rank adds 2 x 24 x 0.125 x 1.5)
    assert bool((y[ids == 1] == want).all())
