"""The 8-bit norm where products x w leave fp32's normal numbers: codes of the definition, with products rounded to
multiples of 2^-149.

Products of 16-bit values are one fp32 value, others the sum of two (the rounded product and what it leaves, each to
2^-149); both are computed here from the 64-bit product, which is exact (at most 24 + 24 bits).
"""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3, I8 = torch.float8_e4m3fn, torch.int8


def codes_of(x, w, dtype, group):
    """(codes as values, groups' largest products) in 64 bits."""
    rows, cols = x.shape
    p = x.double() * w.double()
    near = p.float().double()
    p = near if x.dtype != F32 and w.dtype != F32 else near + (p - near).float().double()
    width = group or cols
    p = torch.nn.functional.pad(p, (0, -cols % width)).view(rows, -1, width)
    top = p.abs().amax(-1, keepdim=True)
    most = 448.0 if dtype == E4M3 else 127.0
    q = p * most / torch.where(top > 0.0, top, 1.0)
    if dtype == E4M3:
        unit = torch.exp2((torch.frexp(q)[1] - 4).clamp(min=-9).double())
        q = torch.round(q / unit) * unit
    else:
        q = torch.round(q)
    return q.reshape(rows, -1)[:, :cols], top.squeeze(-1)


@pytest.mark.parametrize("cols", [256, 1001, 16386, 100001])
@pytest.mark.parametrize("group", [32, 128, None])
@pytest.mark.parametrize("code", [E4M3, I8])
@pytest.mark.parametrize("types", [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_codes(types, code, group, cols):
    g = torch.Generator(device=DEV).manual_seed(cols)
    rows = 7
    # (the row's scale, from the smallest products to those whose two terms are whole)
    power = torch.tensor([-149.0, -148.5, -147.0, -140.0, -126.0, -110.0, -100.0], device=DEV)
    x = torch.randn(rows, cols, generator=g, device=DEV) * torch.exp2(power / 2).unsqueeze(1)
    w = 2.0 ** -49 * (1.0 + 0.3 * torch.randn(cols, generator=g, device=DEV))
    x = (x * torch.exp2(power / 2 + 49.0).unsqueeze(1)).to(types[0])
    w = w.to(types[1])
    got, scales = ops.rms_norm_8bit(x, w, dtype=code, group=group)
    want, top = codes_of(x, w, code, group)
    assert torch.equal(got.double(), want)
    # (v from the rows' own squares, which eps outweighs)
    v = 1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)
    exact = top * v / (448.0 if code == E4M3 else 127.0)
    # v within 4 units in the last place, top and 1 / M rounded, two products; each to 2^-149
    assert bool(((scales.double() - exact).abs() <= 16 * 2.0 ** -24 * exact + 2.0 ** -148).all())


@pytest.mark.parametrize("code,most", [(E4M3, 448.0), (I8, 127.0)])
@pytest.mark.parametrize("cols", [128, 129, 100001])
def test_one_product_between_the_smallest(code, most, cols):
    """1.49 x 2^-149 is held as 2^-149: the group's largest, with the largest code and its sign."""
    x = torch.zeros(2, cols, device=DEV)
    x[0, 3], x[1, 5] = 1.4921875 * 2.0 ** -100, -1.4921875 * 2.0 ** -100
    w = torch.full((cols,), 2.0 ** -49, device=DEV)
    for a, b in ((x.to(BF16), w.to(BF16)), (x.to(BF16), w), (x, w)):
        for group in (32, None):
            got, _ = ops.rms_norm_8bit(a, b, dtype=code, group=group)
            want = torch.zeros(2, cols, device=DEV)
            want[0, 3], want[1, 5] = most, -most
            assert torch.equal(got.float(), want)


@pytest.mark.parametrize("cols", [128, 1001, 100001])
def test_row_of_zeros(cols):
    """Scale 0; with eps 0 the norm is 0 / 0, and so is the scale."""
    x = torch.zeros(3, cols, device=DEV, dtype=BF16)
    x[1] = 1.0
    w = torch.ones(cols, device=DEV, dtype=BF16)
    for group in (64, None):
        codes, scales = ops.rms_norm_8bit(x, w, dtype=I8, group=group)
        assert not bool(scales[[0, 2]].any()) and not bool(codes[[0, 2]].any())
        codes, scales = ops.rms_norm_8bit(x, w, eps=0.0, dtype=I8, group=group)
        assert bool(scales[[0, 2]].isnan().all()) and bool((codes[1] == 127).all())
        y = ops.rms_norm(x, w, eps=0.0)
        assert bool(y[[0, 2]].isnan().all()) and bool((y[1] == 1.0).all())
