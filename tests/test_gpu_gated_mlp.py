"""The gated feed-forward block and its gradients against the formulas in 64 bits.

Bounds are derived, element by element.  With u = eps / 2 of the operand type and t = k 2^-23 (a
sum of k fp32 terms, each addition off by at most a unit in the last place, with products exact):
  |dG| <= t |x| |W|^T =: a (the same for U), the logistic function's relative error r <= 2^-19
  |dh| <= 1.13 a |U| + (|act(G)| + 1.13 a) a + 2 r |h| + u |h|          (|act'| <= 1.13)
  |d(dG)|, |d(dU)| from the same and one rounding to the operand type (up to 65536 tokens x inter two
  terms of it, within u^2)                                               (|act''| <= 0.8)
  |d(dx)| <= |d both| |W13| + t |both| |W13| + u |dx|, likewise dW13
A result below the type's smallest normal is off by at most half its smallest subnormal.
"""

from __future__ import annotations

import math

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def inputs(tokens, hidden, inter, dtype, seed, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (size * torch.randn(tokens, hidden, generator=g, device=DEV)).to(dtype)
    w = (torch.randn(2 * inter, hidden, generator=g, device=DEV) / math.sqrt(hidden)).to(dtype)
    dh = torch.randn(tokens, inter, generator=g, device=DEV).to(dtype)
    return x, w, dh


def act64(g, activation):
    """act, act' in 64 bits."""
    if activation == "silu":
        s, dc = torch.sigmoid(g), torch.ones_like(g)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        s, dc = torch.sigmoid(c * (g + 0.044715 * g ** 3)), c * (1 + 3 * 0.044715 * g * g)
    return g * s, s + g * s * (1 - s) * dc


def formulas(x, w, dh, activation):
    """h, dx, dW13 and their bounds."""
    f = torch.finfo(x.dtype)
    u, tiny = f.eps / 2, f.smallest_normal * f.eps / 2
    x, w, dh = x.double(), w.double(), dh.double()
    hidden, inter = x.shape[1], w.shape[0] // 2
    t, r = hidden * 2.0 ** -23, 2.0 ** -19
    both = x @ w.t()
    a = t * (x.abs() @ w.abs().t())
    g, up = both.chunk(2, 1)
    ag, au = a.chunk(2, 1)
    act, slope = act64(g, activation)
    eact = 1.13 * ag + 2 * r * act.abs()
    h = act * up
    eh = eact * (up.abs() + au) + act.abs() * au + u * h.abs() + tiny
    dg, du = dh * up * slope, dh * act
    eslope = 0.8 * ag + 4 * r
    edg = dh.abs() * (au * (slope.abs() + eslope) + up.abs() * eslope)
    edu = dh.abs() * eact
    d = torch.cat([dg, du], 1)
    terms = u * u if x.shape[0] * inter <= 65536 else u
    ed = torch.cat([edg, edu], 1) * (1 + u) + terms * d.abs() + tiny
    dx, dw = d @ w, d.t() @ x
    tx, tw = 2 * inter * 2.0 ** -23, x.shape[0] * 2.0 ** -23
    edx = (ed + tx * (d.abs() + ed)) @ w.abs() + u * dx.abs()
    edw = (ed + tw * (d.abs() + ed)).t() @ x.abs() + u * dw.abs()
    return (h, dx, dw), (eh, edx * (1 + u) + tiny, edw * (1 + u) + tiny)


def near(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (
        f"off by {(off / bound).max().item():.3g} bounds; max {off.max().item():.3g}")


def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


SHAPES = [(1, 8, 8), (1, 2048, 768), (2, 64, 24), (3, 1000, 712), (4, 264, 8), (5, 8, 8),
          (5, 72, 40), (6, 24, 1000), (8, 512, 256), (150, 8, 16),
          (9, 128, 136), (17, 264, 200), (64, 2048, 768), (127, 320, 128), (128, 64, 128),
          (129, 4096, 264), (333, 1000, 712), (700, 136, 1032), (1500, 640, 520),
          # split reductions: of the forward pass, dx and dW
          (20, 4104, 72), (9, 2048, 2056), (2200, 72, 40), (4100, 264, 136),
          # pairs of SMs: the forward pass, dx and dW, rows past the last pair tile
          (1100, 776, 2184), (1100, 4360, 392), (1057, 2312, 1032)]


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hidden,inter", SHAPES)
def test_forward(tokens, hidden, inter, dtype, activation):
    x, w, dh = inputs(tokens, hidden, inter, dtype, seed=tokens + inter)
    st = status()
    h = ops.gated_mlp(x, w, activation=activation, status=st)
    want, bound = formulas(x, w, dh, activation)
    near(h, want[0], bound[0])
    assert int(st) == 0


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hidden,inter", SHAPES)
def test_gradients(tokens, hidden, inter, dtype, activation):
    x, w, dh = inputs(tokens, hidden, inter, dtype, seed=7 * tokens + inter)
    x.requires_grad_(True)
    w.requires_grad_(True)
    st = status()
    h = ops.gated_mlp(x, w, activation=activation, status=st)
    h.backward(dh)
    want, bound = formulas(x.detach(), w.detach(), dh, activation)
    for got, e, b in zip((h.detach(), x.grad, w.grad), want, bound):
        near(got, e, b)
    assert int(st) == 0
    # the recorded forward pass gives the plain one's values
    with torch.no_grad():
        assert torch.equal(ops.gated_mlp(x, w, activation=activation), h)


def test_gradient_against_differences():
    """dx along a direction against the central difference of sum(h * dh) in 64 bits."""
    x, w, dh = inputs(40, 96, 72, torch.float16, seed=3)
    for activation in ("silu", "gelu_tanh"):
        xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        ops.gated_mlp(xr, wr, activation=activation).backward(dh)

        def loss(a, b):
            g, up = (a @ b.t()).chunk(2, 1)
            return float((act64(g, activation)[0] * up * dh.double()).sum())

        for leaf, grad in ((0, xr.grad), (1, wr.grad)):
            v = torch.randn_like((x, w)[leaf].double())
            step = 1e-5
            lo, hi = [x.double(), w.double()], [x.double(), w.double()]
            lo[leaf], hi[leaf] = lo[leaf] - step * v, hi[leaf] + step * v
            slope = (loss(*hi) - loss(*lo)) / (2 * step)
            _, bound = formulas(x, w, dh, activation)
            # the entries' bounds summed, and the difference's own error (third derivatives of
            # order 1 over a step of 1e-5: far below)
            tol = float((bound[1 + leaf] * v.abs()).sum()) + 1e-6 * abs(slope) + 1e-6
            assert abs(float((grad.double() * v).sum()) - slope) <= tol


@pytest.mark.parametrize("needs", [(True, False), (False, True)])
def test_one_gradient_only(needs):
    x, w, dh = inputs(65, 128, 64, torch.bfloat16, seed=4)
    x.requires_grad_(needs[0])
    w.requires_grad_(needs[1])
    ops.gated_mlp(x, w).backward(dh)
    want, bound = formulas(x.detach(), w.detach(), dh, "silu")
    for leaf, k, n in ((x, 1, needs[0]), (w, 2, needs[1])):
        assert (leaf.grad is not None) == n
        if n:
            near(leaf.grad, want[k], bound[k])


def test_extreme_projections():
    """Projections far out on both sides, and rows of infinities: other rows keep their values."""
    x, w, dh = inputs(32, 64, 32, torch.bfloat16, seed=6, size=1000.0)
    for activation in ("silu", "gelu_tanh"):
        xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        h = ops.gated_mlp(xr, wr, activation=activation)
        h.backward(dh)
        want, bound = formulas(x, w, dh, activation)
        for got, e, b in zip((h.detach(), xr.grad, wr.grad), want, bound):
            near(got, e, b)
        y = x.clone()
        y[3, 5], y[9, 0] = math.inf, math.nan
        got = ops.gated_mlp(y, w, activation=activation)
        keep = [i for i in range(32) if i not in (3, 9)]
        assert torch.equal(got[keep], h.detach()[keep])
        assert bool(torch.isnan(got[9]).all())


def test_no_tokens():
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    w = torch.randn(48, 64, device=DEV).bfloat16().requires_grad_(True)
    h = ops.gated_mlp(x, w)
    assert h.shape == (0, 24)
    h.backward(torch.empty_like(h))
    assert x.grad.shape == (0, 64) and torch.count_nonzero(w.grad) == 0


def test_views_dimensions_and_broadcast_gradients():
    x, w, dh = inputs(60, 128, 64, torch.bfloat16, seed=8)
    wide = torch.randn(60, 131, device=DEV).bfloat16()
    wide[:, 3:] = x
    want = ops.gated_mlp(x, w)
    assert torch.equal(ops.gated_mlp(wide[:, 3:], w), want)
    assert torch.equal(ops.gated_mlp(x.view(3, 20, 128), w), want.view(3, 20, 64))
    assert torch.equal(ops.gated_mlp(x[7], w), ops.gated_mlp(x[7:8], w)[0])
    assert ops.gated_mlp(x.view(3, 20, 128)[:0], w).shape == (0, 20, 64)
    assert torch.equal(ops.gated_mlp(x.t().contiguous().t(), w.t().contiguous().t()), want)
    # an input shared by every row: its gradient is the rows' sum, in the input's type
    one = x[:1].clone().requires_grad_(True)
    ops.gated_mlp(one.expand(60, 128), w).backward(dh)
    rows = x[:1].clone().expand(60, 128).contiguous().requires_grad_(True)
    ops.gated_mlp(rows, w).backward(dh)
    f = torch.finfo(torch.bfloat16)
    bound = 60 * f.eps * rows.grad.double().abs().sum(0, keepdim=True)
    assert bool(((one.grad.double() - rows.grad.double().sum(0, keepdim=True)).abs()
                 <= bound).all())
    # a gradient that comes in expanded, as from sum()
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    ops.gated_mlp(a, w).sum().backward()
    ops.gated_mlp(b, w).backward(torch.ones_like(want))
    assert torch.equal(a.grad, b.grad)


def test_repeatable_streams_and_graphs():
    x, w, dh = inputs(300, 512, 384, torch.bfloat16, seed=9)

    def step():
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        h = ops.gated_mlp(a, b)
        return (h.detach(), *torch.autograd.grad(h, (a, b), dh))

    want = step()
    for got, e in zip(step(), want):
        assert torch.equal(got, e)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for g, e in zip(got, want):
        assert torch.equal(g, e)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(inputs(300, 512, 384, torch.bfloat16, seed=10)[0])
    graph.replay()
    for g, e in zip(out, step()):
        assert torch.equal(g, e)


def test_second_derivative_is_refused():
    x, w, _ = inputs(4, 16, 8, torch.bfloat16, seed=1)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(ops.gated_mlp(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_of_few_values_are_rounded_once(dtype):
    """Few tokens and features: the gradients' error is that of rounding the exact gradients (half a
    unit in the last place at most), not more, in the 2-norm too."""
    x, w, dh = inputs(2, 136, 192, dtype, seed=21)
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    ops.gated_mlp(xr, wr, activation="gelu_tanh").backward(dh)
    want, _ = formulas(x, w, dh, "gelu_tanh")
    for got, e in ((xr.grad, want[1]), (wr.grad, want[2])):
        once = (e.to(dtype).double() - e).norm()
        assert float((got.double() - e).norm()) <= 1.1 * float(once)


def test_calls_at_once_on_two_streams():
    """Products of different sizes and the two kinds of gradients in flight together, many times."""
    sets = []
    for k, (tokens, hidden, inter) in enumerate([(1100, 776, 2184), (300, 512, 384)]):
        x, w, dh = inputs(tokens, hidden, inter, torch.bfloat16, seed=30 + k)
        x.requires_grad_(True)
        w.requires_grad_(True)

        def step(x=x, w=w, dh=dh):
            h = ops.gated_mlp(x, w)
            return (h.detach(), *torch.autograd.grad(h, (x, w), dh))

        sets.append((step, step(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for step, _, stream in sets:
            with torch.cuda.stream(stream):
                got.append(step())
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for a, b in zip(outs, sets[i % 2][1]):
            assert torch.equal(a, b)
