"""fp16 gradients of the gated block where the gradients of its projections, dG = dh U act'(G) and
dU = dh act(G), lie far outside fp16's range of full precision while dx and dW13 do not: a scaled loss, a
mean over many tokens, tokens far apart.

Bounds, element by element, with u = 2^-11, t = k 2^-23 for a sum of k terms, r = 2^-19 for the logistic
function:
  |d(dG)|, |d(dU)| from the projections' error a = t |x| |W|^T as for ordinary sizes (|act'| <= 1.13,
  |act''| <= 0.8), then the 16-bit form's: u of itself (u^2 with two terms, up to 65536 values), or, with
  the largest of the token (for dx) or feature (for dW13) at 2^14 to 2^15 and a subnormal step of 2^-24, at
  least 2^-25 / 2^14 = 2^-39 of that largest;
  |d(dx)| <= |d both| |W13| + t |both| |W13| + u |dx| + 2^-25 (half a subnormal step), likewise dW13.
A result beyond 65504 by more than its bound is an infinity of its sign.
"""

from __future__ import annotations

import math

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def act64(g, activation):
    if activation == "silu":
        s, dc = torch.sigmoid(g), torch.ones_like(g)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        s, dc = torch.sigmoid(c * (g + 0.044715 * g ** 3)), c * (1 + 3 * 0.044715 * g * g)
    return g * s, s + g * s * (1 - s) * dc


def formulas(x, w, dh, activation):
    """dx, dW13, their bounds, and [dG dU]."""
    u, r = 2.0 ** -11, 2.0 ** -19
    x, w, dh = x.double(), w.double(), dh.double()
    hidden, inter = x.shape[1], w.shape[0] // 2
    g, up = (x @ w.t()).chunk(2, 1)
    ag, au = (hidden * 2.0 ** -23 * (x.abs() @ w.abs().t())).chunk(2, 1)
    act, slope = act64(g, activation)
    d = torch.cat([dh * up * slope, dh * act], 1)
    eslope = 0.8 * ag + 4 * r
    ed = torch.cat([dh.abs() * (au * (slope.abs() + eslope) + up.abs() * eslope),
                    dh.abs() * (1.13 * ag + 2 * r * act.abs())], 1)
    ed = ed * (1 + u) + (u * u if x.shape[0] * inter <= 65536 else u) * d.abs()
    top = d.abs() + ed
    dx, dw = d @ w, d.t() @ x
    tx, tw = 2 * inter * 2.0 ** -23, x.shape[0] * 2.0 ** -23
    ex = (ed + 2.0 ** -39 * top.amax(1, keepdim=True) + tx * top) @ w.abs()
    ew = (ed + 2.0 ** -39 * top.amax(0) + tw * top).t() @ x.abs()
    return (dx, dw), (ex * (1 + u) + u * dx.abs() + 2.0 ** -25,
                      ew * (1 + u) + u * dw.abs() + 2.0 ** -25), d


def near(got, want, bound, share):
    """Within the bound where fp16 holds the result (at least `share` of it), else an infinity."""
    got, size = got.double(), want.abs()
    fits = size + bound < 65504
    assert int(fits.sum()) >= share * fits.numel()
    off = (got - want).abs()[fits]
    assert bool((off <= bound[fits]).all()), f"off by {(off / bound[fits]).max().item():.3g} bounds"
    over = size - bound > 65536
    assert torch.equal(got[over], torch.copysign(torch.full_like(got, math.inf), want)[over])


def gradients(x, w, dh, activation):
    x, w = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    h = ops.gated_mlp(x, w, activation=activation, status=status)
    got = torch.autograd.grad(h, (x, w), dh)
    assert int(status) == 0
    return got


def inputs(tokens, hidden, inter, seed, x_size=1.0, w_size=1.0, dh_size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def make(rows, cols, size):
        return (size * torch.randn(rows, cols, generator=g, device=DEV)).half()

    return (make(tokens, hidden, x_size), make(2 * inter, hidden, w_size / math.sqrt(hidden)),
            make(tokens, inter, dh_size))


# two-term sizes, tiles of each kind, split reductions of either gradient, pairs of SMs, and one whose two
# forms of [dG dU] (over 16 MB each) take the same place one behind the other
SHAPES = [(1, 64, 24), (2, 136, 192), (9, 128, 136), (20, 4104, 72), (333, 1000, 712), (2200, 72, 40),
          (4100, 264, 136), (700, 136, 1032), (1100, 776, 2184), (2300, 264, 2056)]


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("tokens,hidden,inter", SHAPES)
def test_scaled_loss(tokens, hidden, inter, activation):
    """dh about 2^12 and projections of 2^3: |dG| goes past 65504, dx (weights of 2^-4) and, in the
    second half, dW13 (activations of 2^-8) do not."""
    for sizes, part in (((2.0 ** 7, 2.0 ** -4), 0), ((2.0 ** -8, 2.0 ** 11), 1)):
        x, w, dh = inputs(tokens, hidden, inter, tokens + inter, *sizes, 2.0 ** 12)
        want, bound, d = formulas(x, w, dh, activation)
        if tokens * inter > 1000:
            assert bool((d.abs() > 65504).any())
        got = gradients(x, w, dh, activation)
        assert bool(torch.isfinite(want[part]).all())
        near(got[part], want[part], bound[part], 0.999)
        near(got[1 - part], want[1 - part], bound[1 - part], 0.0)


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("tokens,hidden,inter", SHAPES)
def test_mean_over_many_tokens(tokens, hidden, inter, activation):
    """dh about 2^-16: most of dG is subnormal or zero in fp16; weights of 2^6, or activations of 2^6,
    bring the gradients back to ordinary size."""
    for sizes, part in (((2.0 ** -6, 2.0 ** 6), 0), ((2.0 ** 6, 2.0 ** -6), 1)):
        x, w, dh = inputs(tokens, hidden, inter, 3 * tokens + inter, *sizes, 2.0 ** -16)
        want, bound, _ = formulas(x, w, dh, activation)
        got = gradients(x, w, dh, activation)
        near(got[part], want[part], bound[part], 1.0)
        near(got[1 - part], want[1 - part], bound[1 - part], 1.0)


@pytest.mark.parametrize("tokens,hidden,inter", [(12, 64, 64), (333, 1000, 712), (1100, 776, 2184)])
def test_tokens_far_apart(tokens, hidden, inter):
    """Tokens from 2^-14 to 2^10 in one batch, one far above them, and empty ones."""
    x, w, dh = inputs(tokens, hidden, inter, 5)
    size = torch.exp2((torch.arange(tokens, device=DEV) % 25) - 14.0).unsqueeze(1)
    dh = (dh.float() * size).half()
    dh[3], dh[5], x[6] = 16384.0, 0.0, 0.0
    x[3] *= 64
    got = gradients(x, w, dh, "silu")
    want, bound, _ = formulas(x, w, dh, "silu")
    near(got[0], want[0], bound[0], 0.5)
    near(got[1], want[1], bound[1], 0.0)  # the large token weighs on every feature
    assert torch.count_nonzero(got[0][5]) == 0
    dh[3, :2], dh[3, 3:] = 0.0, 0.0       # now on one
    got = gradients(x, w, dh, "silu")
    want, bound, _ = formulas(x, w, dh, "silu")
    for k in (0, 1):
        near(got[k], want[k], bound[k], 0.5)


def test_not_finite():
    """A token with an infinite or NaN gradient: dx of the others is what it is without it, and a feature
    with one leaves the other features' weight gradients as they are."""
    x, w, dh = inputs(300, 200, 136, 6)
    dx, dw = gradients(x, w, dh, "silu")
    bad = dh.clone()
    bad[7, 3], bad[9, 100] = math.inf, math.nan
    gx, gw = gradients(x, w, bad, "silu")
    keep = [i for i in range(300) if i not in (7, 9)]
    assert torch.equal(gx[keep], dx[keep])
    assert not bool(torch.isfinite(gx[[7, 9]]).any())
    rows = [i for i in range(272) if i % 136 not in (3, 100)]
    assert torch.equal(gw[rows], dw[rows])
    assert not bool(torch.isfinite(gw[[3, 100, 139, 236]]).any())


@pytest.mark.parametrize("tokens,hidden,inter", [(333, 1000, 712), (2300, 264, 2056)])
@pytest.mark.parametrize("needs", [(True, False), (False, True)])
def test_one_gradient_only(needs, tokens, hidden, inter):
    x, w, dh = inputs(tokens, hidden, inter, 7, dh_size=2.0 ** -10)
    both = gradients(x, w, dh, "gelu_tanh")
    x.requires_grad_(needs[0])
    w.requires_grad_(needs[1])
    ops.gated_mlp(x, w, activation="gelu_tanh").backward(dh)
    for leaf, want, n in ((x, both[0], needs[0]), (w, both[1], needs[1])):
        assert (leaf.grad is not None) == n
        assert not n or torch.equal(leaf.grad, want)


def test_captured_and_repeated():
    x, w, dh = inputs(300, 512, 384, 8, dh_size=2.0 ** -16)

    def step():
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        return torch.autograd.grad(ops.gated_mlp(a, b), (a, b), dh)

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    dh.copy_(inputs(300, 512, 384, 9, dh_size=2.0 ** 9)[2])
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))
