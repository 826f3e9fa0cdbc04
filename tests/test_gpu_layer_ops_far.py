"""Norm, balance loss and adapters over more than 2^31 elements: the last rows against the formula in 64 bits
or a call of their own, whose offsets are small."""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
E = 2.0 ** -24


def normal(*shape, dtype):
    g = torch.Generator(device=DEV).manual_seed(11)
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=g)


@pytest.mark.parametrize("rows,cols", [(2_150_001, 1001), (530_001, 4096)])
def test_norm(rows, cols):
    assert rows * cols > 2 ** 31
    x, w = normal(rows, cols, dtype=torch.float16), normal(cols, dtype=torch.float16)
    last = slice(rows - 64, rows)
    mine = x[last].clone()
    y = ops.rms_norm(x, w)
    # (not the bits of a call on these rows alone: it may take the sum of squares in another order.)  The
    # sum in chains of at most 32 and 10 more, halved by the root: v within 26 e; y's products and rounding
    s, f = mine.double(), w.double()
    v = torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6)
    want = s * v * f
    assert bool(((y[last].double() - want).abs() <=
                 (29 * E + 2.0 ** -11) * want.abs() + 2.0 ** -25).all())
    for group in (None, 64):
        codes, scales = ops.rms_norm_8bit(x, w, group=group)
        few, few_scales = ops.rms_norm_8bit(mine, w, group=group)
        assert torch.equal(codes[last].view(torch.uint8), few.view(torch.uint8))
        # (a sum's order may be another's: each within (32 / 2 + 14) e of the definition's)
        assert bool(((scales[last] - few_scales).abs() <= 60 * E * few_scales).all())
    back = ops.dequantize_8bit(codes, scales, group=64, dtype=torch.float16)
    want = codes[last].double() * scales[last].double().repeat_interleave(64, 1)[:, :cols]
    assert torch.equal(back[last], want.float().half())
    del codes, scales, back
    x.requires_grad_()
    dx, = torch.autograd.grad(ops.rms_norm(x, w), x, y)
    mine.requires_grad_()
    few, = torch.autograd.grad(ops.rms_norm(mine, w), mine, y[last].clone())
    # of y in place of dy: dx = v (w y - s v^2 mean(w y s)), rounded once by each call; each call's fp32
    # roundings at most (26 + 7) e of the first term, (45 + 3 26 + 6 + 3) e of the second's terms
    up = f * y[last].double()
    size = v * up.abs() + s.abs() * v ** 3 * (up * s).abs().mean(-1, keepdim=True)
    assert bool(((dx[last].double() - few.double()).abs() <=
                 2.0 ** -10 * few.double().abs() + 264 * E * size + 2.0 ** -24).all())


def test_balance_loss():
    tokens, experts = 16_900_001, 128
    assert tokens * experts > 2 ** 31
    x = normal(tokens, experts, dtype=torch.bfloat16).requires_grad_()
    ids = (torch.arange(tokens, device=DEV) * 7 % 131).to(torch.int32).view(tokens, 1)  # some outside
    loss, counts = ops.balance_loss(x, ids)
    c = torch.bincount(ids.view(-1).long(), minlength=131)[:experts]
    assert torch.equal(counts.long().view(-1), c)
    total = torch.zeros(experts, dtype=torch.float64, device=DEV)
    for part in x.detach().split(1 << 20):
        total += torch.softmax(part.double(), -1).sum(0)
    want = experts / tokens ** 2 * float((c.double() * total).sum())
    # a token's probabilities within 2^-20, sums of up to tokens / 592 / 8 / 4 of them in fp32: their roundings
    # are at most (that + 50) e of the sum
    assert abs(float(loss.detach()) - want) <= (2.0 ** -20 + (tokens / 592 / 32 + 50) * E) * want
    grad, = torch.autograd.grad(loss, x)
    last = slice(tokens - 64, tokens)
    p = torch.softmax(x.detach()[last].double(), -1)
    a = experts / tokens ** 2 * c.double()
    exact = p * (a - (p * a).sum(-1, keepdim=True))
    # counts less their mean stay below 2^18: the difference's terms
    spread = experts / tokens ** 2 * (c.double() - tokens // experts).abs().max()
    bound = 2.0 ** -8 * exact.abs() + p * spread * 2.0 ** -17 + 2.0 ** -133
    assert bool(((grad[last].double() - exact).abs() <= bound).all())


@pytest.mark.parametrize("inner,outer", [(2048, 64), (64, 2048)])
def test_adapted_linear(inner, outer):
    tokens, adapters, rank = 1_050_000, 3, 16
    assert tokens * max(inner, outer) > 2 ** 31
    x, w = normal(tokens, inner, dtype=torch.bfloat16), normal(outer, inner, dtype=torch.bfloat16)
    a, b = normal(adapters, rank, inner, dtype=torch.bfloat16), normal(adapters, outer, rank,
                                                                       dtype=torch.bfloat16)
    ids = (torch.arange(tokens, device=DEV) // 1000 % 4 - 1).to(torch.int32)
    y = ops.adapted_linear(x, w, a, b, ids)
    last = slice(tokens - 64, tokens)
    for t in range(tokens - 64, tokens):
        xt, i = x[t].double(), int(ids[t])
        want, terms = w.double() @ xt, w.double().abs() @ xt.abs()
        if i >= 0:
            z = a[i].double() @ xt
            want = want + b[i].double() @ z
            terms = terms + b[i].double().abs() @ (a[i].double().abs() @ xt.abs())
        # the result's rounding, z's two 16-bit terms 2^-16, fp32 sums of inner + 2 rank terms
        bound = 2.0 ** -8 * want.abs() + (2.0 ** -16 + (inner + 2 * rank) * E) * terms
        assert bool(((y[t].double() - want).abs() <= bound).all())
    assert y[last].shape == (64, outer)
