"""Gates far out on the negative side, where the logistic function is as small as fp32 holds: products of
one gate value and one factor (every other entry of the rows and weights is 0), so that the sums are exact
and the error is the activation's and the roundings'.

With e = (2 + 1.2 |c|) 2^-23 the error of e^c and 2^-21 that of the quotient and products, relative, a
value is off by at most 2 (e + 2^-21) of itself and, where the logistic function s is subnormal, by
(3 |g| + 1) |u| 2^-149: the fast exponential is rounded to a step of 2^-149, the fast quotient is within 2
units in the last place, which are such steps, and s enters as g s u, the product g s being rounded to a
step once more.  Then come the roundings: to bf16, whose values lie 2^-7 apart at 1, 2^-8 and half a
subnormal step, 2^-134; the intermediate value of the MXFP4 experts 2^-9 and 2^-137.
"""

from __future__ import annotations

import math

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def gates(tokens):
    """bf16 values: steps of a half from -127.5 on, finer ones around -10.4 (gelu's edge), some up to 40."""
    g = torch.cat([torch.arange(-255, -100) / 2, torch.arange(-200, -130) / 16,
                   torch.arange(-40, 41).float()])
    g = g.repeat(-(-tokens // g.numel()))[:tokens]
    assert torch.equal(g.bfloat16().float(), g.float())
    return g.to(DEV).double()


def act64(g, activation):
    """act, act', c and the relative error of the logistic function."""
    k = 2 * math.sqrt(2 / math.pi)
    c = g if activation == "silu" else k * (g + 0.044715 * g ** 3)
    dc = torch.ones_like(g) if activation == "silu" else k * (1 + 3 * 0.044715 * g * g)
    s = torch.sigmoid(c)
    rel = 2 * ((2 + 1.2 * c.abs()) * 2.0 ** -23 + 2.0 ** -21)
    if activation == "gelu_tanh":  # c itself is rounded: a few units in its last place
        rel = rel + 4 * c.abs() * 2.0 ** -23
    return g * s, s + g * s * (1 - s) * dc, rel


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("tokens,hidden,inter", [(1, 64, 8), (4, 64, 8), (306, 64, 8), (306, 2056, 8),
                                                 (1100, 776, 2184)])
def test_gated(tokens, hidden, inter, activation):
    g = gates(tokens) if tokens > 4 else gates(306)[78:78 + tokens]  # -88.5 on
    x = torch.zeros(tokens, hidden, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(2 * inter, hidden, dtype=torch.bfloat16, device=DEV)
    x[:, 0], x[:, 1] = g.bfloat16(), 2.0 ** 20
    w[:inter, 0], w[inter:, 1] = 1.0, 2.0 ** 20
    up = 2.0 ** 40
    act, slope, rel = act64(g, activation)
    x.requires_grad_(True)
    h = ops.gated_mlp(x, w, activation=activation)
    off = (h.detach().double() - (act * up).unsqueeze(1)).abs()
    bound = (rel + 2.0 ** -8) * (act * up).abs() + (3 * g.abs() + 1) * up * 2.0 ** -149 + 2.0 ** -134
    assert bool((off <= bound.unsqueeze(1)).all()), float((off / bound.unsqueeze(1)).max())
    (dx,) = torch.autograd.grad(h, x, torch.ones_like(h))
    # dx[:, 0] = inter * dG, dx[:, 1] = 2^20 inter * dU; [dG dU] and dx are rounded, sums of inter terms;
    # act' = s + g s (1 - s) c': its two parts' errors add up
    s = torch.sigmoid(g if activation == "silu" else
                      2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
    parts = s.abs() + (slope - s).abs()
    terms = 2.0 ** -16 if tokens * inter <= 65536 else 2.0 ** -8
    r = 2.0 ** -8 + 1.01 * terms + inter * 2.0 ** -23
    dg, du = inter * up * slope, inter * 2.0 ** 20 * act
    for got, want, size, more in (
            (dx[:, 0], dg, inter * up * parts, inter * up * (1 + g.abs()) * 50 * 2.0 ** -149),
            (dx[:, 1], du, du.abs(), inter * 2.0 ** 20 * (g.abs() * 2.0 ** -149 + 2.0 ** -126))):
        bound = r * want.abs() + 3 * rel * size + more + inter * 2.0 ** -126
        off = (got.double() - want).abs()
        assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("tokens,experts", [(60, 4), (306, 16), (306, 4)])
def test_experts(tokens, experts):
    """A few routes, decode and prefill."""
    hidden, inter = 256, 128
    g = gates(306)[50:50 + tokens] if tokens <= 60 else gates(tokens)
    w13 = torch.zeros(experts, 2 * inter, hidden, device=DEV)
    w13[:, :inter, 0], w13[:, inter:, 1] = 1.0, 2.0 ** 10
    w2 = torch.zeros(experts, hidden, inter, device=DEV)
    w2[:, :, 5] = 1.0
    (c13, s13), (c2, s2) = ops.quantize_mxfp4(w13), ops.quantize_mxfp4(w2)
    x = torch.zeros(tokens, hidden, dtype=torch.bfloat16, device=DEV)
    x[:, 0], x[:, 1] = g.bfloat16(), 2.0 ** 10
    ids = torch.arange(tokens, dtype=torch.int32, device=DEV).remainder(experts).unsqueeze(1)
    y = ops.fused_experts_mxfp4(x, torch.ones(tokens, 1, device=DEV), ids, c13,
                                ops.tile_mxfp4_scales(s13), c2, ops.tile_mxfp4_scales(s2))
    act, _, rel = act64(g, "silu")
    want = act * 2.0 ** 20
    # prefill holds route outputs within 2^-14 of the largest (here all are equal), at least 2^-127
    bound = ((rel + 2.0 ** -8 + 1.01 * 2.0 ** -9 + 2.0 ** -14) * want.abs()
             + (3 * g.abs() + 1) * 2.0 ** 20 * 2.0 ** -149 + 2.0 ** -126)
    off = (y.double() - want.unsqueeze(1)).abs()
    assert bool((off <= bound.unsqueeze(1)).all()), float((off / bound.unsqueeze(1)).max())
