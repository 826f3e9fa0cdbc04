"""The balance loss, its counts and its gradient against the formula in 64 bits.

Bounds are derived.  With e = 2^-24: a score's relative error is that of an exponential (2^-21), of a sum
of at most 1024 terms of one sign in chains of 37 and of two more roundings: ep = 2^-21 + 44 e (sigmoid:
the exponential and its sum enter once more: twice that).  A column's sum over tokens adds T / 1000 + 40
roundings of fp32 at most (8 warps a block, 148 blocks a group of many tokens; a warp's tokens of a block
of 64 otherwise).  The gradient is size p (c - p c): p is off by ep, the dot by (ep + 40 e) sum p |c|,
with c less its mean, and the result is rounded to the type.
"""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -24


def inputs(groups, tokens, experts, top_k, dtype, seed, size=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = size * torch.randn(groups, tokens, experts, generator=g, device=DEV)
    x = (x + torch.randn(groups, 1, experts, generator=g, device=DEV)).to(dtype)
    ids = x.float().topk(top_k, -1).indices.int()
    mask = torch.rand(groups, tokens, generator=g, device=DEV) < 0.7
    dloss = tokens * (0.5 + torch.rand(groups, generator=g, device=DEV))
    return x, ids, mask, dloss


def formula(x, ids, mask, dloss, scoring):
    """((loss, counts, gradient), (bound of the loss, bound of the gradient))"""
    f = torch.finfo(x.dtype)
    u, tiny = f.eps / 2, f.smallest_normal * f.eps / 2
    n, t, e = x.shape
    k = ids.shape[-1]
    mask = torch.ones(n, t, dtype=torch.bool, device=DEV) if mask is None else mask
    x = torch.where(mask.unsqueeze(-1), x.double(), 0.0)
    if scoring == "softmax":
        p = torch.softmax(x, -1)
        ep = 2.0 ** -21 + 44 * E
        slope = torch.ones_like(p)
    else:
        low = x.amax(-1, keepdim=True) < -600.0
        p = torch.where(low, torch.softmax(x, -1),
                        torch.sigmoid(x) / torch.sigmoid(x).sum(-1, keepdim=True))
        ep = 2.0 ** -20 + 88 * E
        slope = torch.sigmoid(-x)
    p = torch.where(mask.unsqueeze(-1), p.nan_to_num(nan=0.0) if bool(
        (x == -float("inf")).all(-1).any()) else p, 0.0)
    there = mask.unsqueeze(-1) & (ids >= 0) & (ids < e)
    counts = torch.zeros(n, e + 1, dtype=torch.int64, device=DEV)
    counts.scatter_add_(1, torch.where(there, ids.long(), e).reshape(n, -1),
                        torch.ones(n, t * k, dtype=torch.int64, device=DEV))
    counts = counts[:, :e]
    valid = mask.sum(-1)
    size = e / (k * valid.clamp(min=1).double() ** 2)
    loss = size * (counts * p.sum(1)).sum(-1)
    eloss = loss * (ep + (t / 1000 + 48) * E) * (1 + u)
    size = (size * dloss.double()).view(n, 1, 1)
    c = counts.double().unsqueeze(1) - (valid * k / e).view(n, 1, 1).floor()
    dot = (p * c).sum(-1, keepdim=True)
    grad = size * p * (c - dot) * slope
    edot = (p * c.abs()).sum(-1, keepdim=True) * (2 * ep + 40 * E)
    eg = size.abs() * p * slope * ((c - dot).abs() * (2 * ep + 8 * E) + edot) * 1.01
    return (loss, counts.int(), grad), (eloss, eg + u * grad.abs() * 1.01 + tiny)


def near(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (
        f"off by {(off / bound).max().item():.3g} bounds; max {off.max().item():.3g}")


def check(x, ids, mask, dloss, scoring):
    x = x.detach().requires_grad_(True)
    loss, counts = ops.balance_loss(x, ids, scoring=scoring, mask=mask)
    grad, = torch.autograd.grad(loss, x, dloss)
    want, bound = formula(x.detach(), ids, mask, dloss, scoring)
    assert counts.dtype == torch.int32 and torch.equal(counts, want[1])
    near(loss.detach(), want[0], bound[0])
    assert grad.dtype == x.dtype
    near(grad, want[2], bound[1])
    with torch.no_grad():
        plain = ops.balance_loss(x, ids, scoring=scoring, mask=mask)
    assert torch.equal(plain[0], loss.detach()) and torch.equal(plain[1], counts)
    return loss.detach(), counts, grad


SHAPES = [(1, 1, 2, 1), (1, 1, 8, 8), (2, 3, 5, 2), (1, 63, 8, 2), (3, 65, 16, 4), (1, 512, 64, 8),
          (2, 1000, 60, 6), (16, 100, 128, 8), (1, 20000, 128, 8), (4, 700, 256, 8), (2, 300, 160, 3),
          (1, 900, 257, 7), (2, 333, 512, 8), (1, 500, 1000, 4), (1, 400, 1024, 8), (1, 300, 1023, 1),
          (300, 5, 24, 2), (1, 50, 1, 1)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("groups,tokens,experts,top_k", SHAPES)
def test_loss_counts_and_gradient(groups, tokens, experts, top_k, dtype, scoring):
    x, ids, mask, dloss = inputs(groups, tokens, experts, top_k, dtype, tokens + experts)
    check(x, ids, None, dloss, scoring)
    check(x, ids, mask, dloss, scoring)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("experts", [64, 100])
def test_left_out_tokens(experts, dtype, scoring):
    """What stands in left-out tokens does not matter; a group of none has a loss of 0."""
    x, ids, mask, dloss = inputs(4, 200, experts, 4, dtype, 7)
    mask[2] = False
    mask[3] = False
    mask[3, 199] = True
    loss, counts, grad = check(x, ids, mask, dloss, scoring)
    assert float(loss[2]) == 0.0 and not counts[2].any() and not grad[2].any()
    low = torch.finfo(dtype).min
    for junk in (float("nan"), float("inf"), -float("inf"), low):
        y = torch.where(mask.unsqueeze(-1), x, junk)
        i = torch.where(mask.unsqueeze(-1), ids, 3)
        got = check(y, i, mask, dloss, scoring)
        assert all(torch.equal(a, b) for a, b in zip(got, (loss, counts, grad)))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_experts_that_cannot_be_chosen(dtype):
    """Logits of -inf or the type's lowest value; a row of nothing else has no scores."""
    x, ids, _, dloss = inputs(2, 100, 64, 4, dtype, 5)
    for low in (-float("inf"), torch.finfo(dtype).min):
        y = x.clone()
        y[:, :, ::3] = low
        _, _, grad = check(y, ids, None, dloss, "softmax")
        assert not grad[:, :, ::3].any()
        check(y, ids, None, dloss, "sigmoid")
    y = x.clone()
    y[0, 5] = -float("inf")
    for scoring in ("softmax", "sigmoid"):
        _, _, grad = check(y, ids, None, dloss, scoring)
        assert not grad[0, 5].any()
    y[0, 5] = torch.finfo(dtype).min  # even scores
    check(y, ids, None, dloss, "softmax")
    # a NaN that is not left out is not hidden
    y[1, 7, 3] = float("nan")
    loss, _ = ops.balance_loss(y, ids)
    assert bool(loss[1].isnan()) and not bool(loss[0].isnan())


@pytest.mark.parametrize("shift", [-500.0, -88.0, -60.0, -29.0, 40.0, 200.0])
def test_far_logits(shift):
    x, ids, _, dloss = inputs(1, 50, 64, 4, F32, 9)
    for scoring in ("softmax", "sigmoid"):
        check(x + shift, ids, None, dloss, scoring)


def test_ids():
    x, ids, mask, dloss = inputs(2, 300, 128, 8, BF16, 3)
    want = check(x, ids, mask, dloss, "softmax")
    for dtype in (torch.int64, torch.int16, torch.uint8):
        got = check(x, ids.to(dtype), mask, dloss, "softmax")
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    far = ids.clone()
    far[:, ::2] = -1
    far[:, 1::4, 0] = 128
    far[0, 0, 0] = 2 ** 31 - 1
    check(x, far, mask, dloss, "softmax")
    far = far.long()
    far[0, 1, 1] = 2 ** 40 + 5
    far[0, 1, 2] = -(2 ** 40)
    check(x, far, mask, dloss, "sigmoid")
    # the same expert for every route
    check(x, torch.full_like(ids, 127), None, dloss, "softmax")
    with pytest.raises(TypeError):
        ops.balance_loss(x, ids.float())


def test_shapes_and_strides():
    x, ids, mask, dloss = inputs(6, 40, 64, 4, F32, 21)
    want = check(x, ids, mask, dloss, "softmax")
    loss, counts = ops.balance_loss(x.view(2, 3, 40, 64), ids.view(2, 3, 40, 4),
                                    mask=mask.view(2, 3, 40))
    assert loss.shape == (2, 3) and counts.shape == (2, 3, 64)
    assert torch.equal(loss.view(6), want[0]) and torch.equal(counts.view(6, 64), want[1])
    one, c = ops.balance_loss(x[1], ids[1], mask=mask[1])
    assert one.shape == () and c.shape == (64,)
    near(one.double(), want[0][1].double(), 8 * E * want[0][1].double())
    # tokens outermost, another group's columns beside them, an odd start
    t = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.balance_loss(t, ids, mask=mask)[0], want[0])
    flat = torch.zeros(x.numel() + 1, device=DEV)
    flat[1:] = x.reshape(-1)
    odd = flat[1:].view_as(x)
    check(odd, ids, mask, dloss, "softmax")
    # broadcast logits, and a gradient through the broadcast
    b = x[0].clone().requires_grad_(True)
    loss, _ = ops.balance_loss(b.expand(6, 40, 64), ids, mask=mask)
    grad, = torch.autograd.grad(loss, b, dloss)
    w, bound = formula(x[:1].expand(6, 40, 64), ids, mask, dloss, "softmax")
    near(grad, w[2].sum(0), bound[1].sum(0) + 6 * E * w[2].abs().sum(0))
    # nothing at all
    for shape in ((0, 40, 64), (3, 0, 64)):
        e = torch.zeros(shape, device=DEV, requires_grad=True)
        loss, counts = ops.balance_loss(e, torch.zeros(*shape[:-1], 4, dtype=torch.int32, device=DEV))
        assert loss.shape == shape[:1] and not loss.any() and not counts.any()
        loss.sum().backward()
        assert e.grad.shape == shape


def test_differences():
    """The gradient against central differences of the formula in 64 bits."""
    x, ids, mask, dloss = inputs(2, 6, 10, 2, F32, 2)
    for scoring in ("softmax", "sigmoid"):
        a = x.clone().requires_grad_(True)
        loss, counts = ops.balance_loss(a, ids, scoring=scoring, mask=mask)
        grad, = torch.autograd.grad(loss, a, dloss)

        def value(v):
            p = torch.softmax(v, -1) if scoring == "softmax" else (
                torch.sigmoid(v) / torch.sigmoid(v).sum(-1, keepdim=True))
            p = p * mask.unsqueeze(-1)
            n = mask.sum(-1).clamp(min=1).double()
            return (10 / (2 * n * n) * (counts * p.sum(1)).sum(-1) * dloss.double()).sum()

        h = 1e-4
        for j in range(x.numel()):
            up, down = x.double(), x.double()
            up.view(-1)[j] += h
            down.view(-1)[j] -= h
            slope = float((value(up) - value(down)) / (2 * h))
            assert abs(slope - float(grad.reshape(-1)[j])) < 1e-5 * (1.0 + abs(slope))


def test_graph_streams_order_and_refusals():
    x, ids, mask, dloss = inputs(3, 2000, 128, 8, BF16, 4)
    a = x.clone().requires_grad_(True)
    loss, counts = ops.balance_loss(a, ids, mask=mask)
    grad, = torch.autograd.grad(loss, a, dloss)
    first = (loss.detach().clone(), counts.clone(), grad.clone())
    del loss, counts, grad
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.balance_loss(x, ids, mask=mask)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other[0], first[0]) and torch.equal(other[1], first[1])
    for _ in range(5):  # the same bits every time
        again = ops.balance_loss(x, ids, mask=mask)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, counts = ops.balance_loss(a, ids, mask=mask)
        grad, = torch.autograd.grad(loss, a, dloss)
    for t in (loss.detach(), counts, grad):
        t.zero_()
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip((loss.detach(), counts, grad), first))

    with pytest.raises(TypeError):
        ops.balance_loss(x.double(), ids)
    with pytest.raises(ValueError):
        ops.balance_loss(x, ids, scoring="sqrtsoftplus")
    with pytest.raises(ValueError):
        ops.balance_loss(x, ids[:, :-1])
    with pytest.raises(ValueError):
        ops.balance_loss(x, ids, mask=mask.float())
    with pytest.raises(ValueError):
        ops.balance_loss(x, ids, mask=mask[:1])
    with pytest.raises(NotImplementedError):
        ops.balance_loss(torch.zeros(2, 1025, device=DEV), torch.zeros(2, 1, dtype=torch.int32,
                                                                       device=DEV))
    loss, _ = ops.balance_loss(a, ids)
    g, = torch.autograd.grad(loss.sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), a)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        with pytest.raises(NotImplementedError):
            ops.balance_loss(dual, ids)


def test_low_sigmoid_rows():
    """Rows whose sigmoids are all small, on both sides of where they become softmaxes."""
    for top in (-10.0, -17.9, -18.1, -29.0, -31.0, -80.0):
        g = torch.Generator(device=DEV).manual_seed(1)
        x = top - 60.0 * torch.rand(1, 300, 96, generator=g, device=DEV)
        x[:, :, 5] = top
        ids = torch.randint(0, 96, (1, 300, 4), generator=g, device=DEV).int()
        dloss = torch.full((1,), 300.0, device=DEV)
        a = x.clone().requires_grad_()
        loss, counts = ops.balance_loss(a, ids, scoring="sigmoid")
        grad, = torch.autograd.grad(loss, a, dloss)
        (want, c, dx), (eloss, edx) = formula(x, ids, None, dloss, "sigmoid")
        assert torch.equal(counts, c)
        near(loss.detach(), want, eloss)
        near(grad, dx, edx)
