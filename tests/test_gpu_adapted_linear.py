"""The projection with adapters against its formula in 64 bits.

Bounds are derived, element by element.  With u = eps / 2 of the type and t(n) = n 2^-23 (a sum of n fp32
terms, each addition off by at most a unit in the last place, with products exact):
  |dz| <= (t(K) + 2^-23) s |x| |A|^T + (u^2 + t(8)) |z|  (the scaling's product, two terms of the type
    above 128 tokens, parts joined), and half of fp16's smallest subnormal
  |dy| <= t(K + 2 rank) (|x| |W|^T + |z| |B|^T) + |dz| |B|^T + u |y|
A result below the type's smallest normal is off by at most half its smallest subnormal.
"""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16 = torch.bfloat16, torch.float16


def inputs(tokens, inner, outer, adapters, rank, dtype, seed, runs=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, size=1.0):
        return (size * torch.randn(*shape, generator=g, device=DEV)).to(dtype)

    x, w = normal(tokens, inner), normal(outer, inner, size=inner ** -0.5)
    a = normal(adapters, rank, inner, size=inner ** -0.5)
    b = normal(adapters, outer, rank, size=rank ** -0.5)
    s = 0.5 + 1.5 * torch.rand(adapters, generator=g, device=DEV)
    if runs == 0:
        ids = torch.randint(-1, adapters, (tokens,), generator=g, device=DEV)
    else:
        cuts = torch.randint(0, tokens, (runs,), generator=g, device=DEV).sort()[0]
        mine = torch.randint(-1, adapters, (runs + 1,), generator=g, device=DEV)
        ids = mine[torch.searchsorted(cuts, torch.arange(tokens, device=DEV), right=True)]
    return x, w, a, b, ids.int(), s


def formula(x, w, a, b, ids, s):
    """(y, its bound) in 64 bits."""
    f = torch.finfo(x.dtype)
    u, tiny = f.eps / 2, f.smallest_normal * f.eps / 2
    tokens, inner = x.shape
    rank = a.shape[1]
    x, w = x.double(), w.double()
    t = 2.0 ** -23
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    extra = torch.zeros_like(y)
    for i in torch.unique(ids).tolist():
        if not 0 <= i < a.shape[0]:
            continue
        rows = (ids == i).nonzero().squeeze(1)
        scale = 1.0 if s is None else float(s[i])
        ai, bi = a[i].double(), b[i].double()
        z = scale * (x[rows] @ ai.t())
        dz = ((inner + 1) * t * scale * (x[rows].abs() @ ai.abs().t())
              + (u * u + 8 * t) * z.abs() + (tiny if f.eps < 2.0 ** -8 else 0.0))
        y[rows] += z @ bi.t()
        size[rows] += z.abs() @ bi.abs().t()
        extra[rows] += dz @ bi.abs().t()
    bound = (inner + 2 * rank) * t * size + extra * (1 + u) + u * y.abs() + tiny
    return y, bound * (1 + u)


def near(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (
        f"off by {(off / bound).max().item():.3g} bounds; max {off.max().item():.3g}")


def check(x, w, a, b, ids, s):
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    y = ops.adapted_linear(x, w, a, b, ids, scaling=s, status=status)
    assert int(status) == 0
    near(y, *formula(x, w, a, b, ids, s))
    return y


SHAPES = [
    # tokens, inner, outer, adapters, rank
    (1, 8, 8, 1, 8), (1, 2048, 4096, 4, 16), (2, 72, 40, 3, 24), (3, 1000, 520, 2, 64),
    (8, 264, 200, 9, 40), (9, 2048, 768, 3, 128), (16, 520, 1032, 20, 8), (16, 4096, 264, 2, 72),
    # tiles: 64, 128 and 256 columns, split reductions, one and several tiles of tokens
    (17, 8, 8, 1, 8), (17, 40, 72, 4, 16), (64, 2048, 4096, 32, 16), (65, 1000, 712, 70, 24),
    (100, 768, 2048, 200, 8), (127, 320, 1000, 3, 128), (128, 4096, 264, 128, 16),
    (129, 264, 136, 5, 56), (256, 1032, 520, 300, 40), (257, 2048, 768, 11, 32),
    (300, 72, 5000, 4, 64), (1000, 2056, 2056, 6, 16), (1500, 136, 4104, 9, 112),
    (2500, 520, 4096, 12, 64), (4200, 256, 2048, 40, 8), (300, 2048, 264, 300, 16),
    (700, 4104, 264, 2, 128), (520, 776, 136, 3, 96), (260, 8, 8, 2, 8),
    # reductions among 3, 5, 6 and 7 blocks
    (128, 1544, 264, 6, 32), (127, 2568, 136, 6, 48), (256, 3112, 136, 3, 16), (128, 3592, 72, 128, 8),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,inner,outer,adapters,rank", SHAPES)
def test_against_formula(tokens, inner, outer, adapters, rank, dtype):
    args = inputs(tokens, inner, outer, adapters, rank, dtype, tokens + inner)
    check(*args)  # every token its own
    args = inputs(tokens, inner, outer, adapters, rank, dtype, tokens + outer, runs=5)
    check(*args)
    check(*args[:5], None)


@pytest.mark.parametrize("tokens", [1, 5, 16, 40, 300])
def test_which_adapter(tokens):
    """None, one for all, one token's, ids outside, and that other adapters' values do not matter."""
    x, w, a, b, _, s = inputs(tokens, 264, 136, 4, 16, BF16, tokens)
    none = torch.full((tokens,), -1, dtype=torch.int32, device=DEV)
    plain = check(x, w, a, b, none, s)
    for ids in (none + 1, none + 4, torch.arange(tokens, device=DEV).int() % 4):
        check(x, w, a, b, ids, s)
    far = none.clone()
    far[::2] = 4
    far[1::3] = 2 ** 31 - 1
    assert torch.equal(check(x, w, a, b, far, s), plain)
    wide = far.long()
    wide[::2] = -(2 ** 40)
    assert torch.equal(check(x, w, a, b, wide, s), plain)
    one = none.clone()
    one[tokens // 2] = 2
    y = check(x, w, a, b, one, s)
    others = torch.arange(tokens, device=DEV) != tokens // 2
    assert torch.equal(y[others], plain[others])
    a2, b2, s2 = a.clone(), b.clone(), s.clone()
    for t in (a2, b2, s2):
        t[:2] = float("nan")
        t[3] = float("inf")
    assert torch.equal(ops.adapted_linear(x, w, a2, b2, one, scaling=s2), y)
    # a token that holds a NaN keeps it to itself
    x2 = x.clone()
    x2[0, 3] = float("nan")
    y2 = ops.adapted_linear(x2, w, a, b, none + 2, scaling=s)
    want = ops.adapted_linear(x, w, a, b, none + 2, scaling=s)
    assert bool(y2[0].isnan().all()) and torch.equal(y2[1:], want[1:])
    # as does an adapter of its own tokens
    if tokens > 1:
        half = none + 1
        half[tokens // 2:] = 2
        a3 = a.clone()
        a3[2, 0, 0] = float("nan")
        y3 = ops.adapted_linear(x, w, a3, b, half, scaling=s)
        assert bool(y3[tokens // 2:].isnan().all())
        assert torch.equal(y3[:tokens // 2], ops.adapted_linear(x, w, a, b, half, scaling=s)[
            :tokens // 2])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,inner", [(8, 264), (50, 264), (50, 4096), (300, 264),
                                          (300, 4096)])
def test_one_requests_broken_adapter(tokens, inner, dtype):
    """Infinities and NaN of an adapter's B reach its own tokens' features alone."""
    x, w, a, b, _, s = inputs(tokens, inner, 136, 3, 24, dtype, tokens)
    ids = torch.arange(tokens, device=DEV).int() % 4 - 1
    want = check(x, w, a, b, ids, s)
    broken = b.clone()
    broken[1, 5, 3] = float("inf")
    broken[1, 70, 23] = float("nan")
    broken[1, 135, 8] = -float("inf")
    y = ops.adapted_linear(x, w, a, broken, ids, scaling=s)
    own = ids == 1
    assert torch.equal(y[~own], want[~own])
    good = torch.ones(136, dtype=torch.bool, device=DEV)
    good[[5, 70, 135]] = False
    assert torch.equal(y[own][:, good], want[own][:, good])
    assert bool(y[own][:, 70].isnan().all())
    z = (x[own].double() @ a[1].double().t())
    assert torch.equal(y[own][:, 5], (z[:, 3] * float("inf")).to(dtype))
    assert torch.equal(y[own][:, 135], (z[:, 8] * -float("inf")).to(dtype))


def test_far_apart_terms():
    """Adapters that outweigh the projection: z keeps two terms' accuracy."""
    for dtype in (BF16, F16):
        for tokens in (4, 50):
            x, w, a, b, ids, s = inputs(tokens, 512, 256, 3, 16, dtype, 5)
            w = torch.zeros_like(w)
            check(x, w, a, (8 * b.float()).to(dtype), ids, 4 * s)


def test_shapes_strides_ids_and_empty():
    x, w, a, b, ids, s = inputs(24, 264, 136, 4, 16, BF16, 1)
    want = ops.adapted_linear(x, w, a, b, ids, scaling=s)
    y = ops.adapted_linear(x.view(2, 3, 4, 264), w, a, b, ids.view(2, 3, 4), scaling=s)
    assert y.shape == (2, 3, 4, 136) and torch.equal(y.view(24, 136), want)
    assert torch.equal(ops.adapted_linear(x, w, a, b, ids.to(torch.int8), scaling=s), want)
    assert torch.equal(ops.adapted_linear(x, w, a, b, ids.long(), scaling=s.double()), want)
    wide = torch.zeros(24, 300, dtype=BF16, device=DEV)
    wide[:, 3:267] = x
    assert torch.equal(ops.adapted_linear(wide[:, 3:267], w, a, b, ids, scaling=s), want)
    assert torch.equal(ops.adapted_linear(x, w.t().contiguous().t(), a,
                                          b.transpose(1, 2).contiguous().transpose(1, 2), ids,
                                          scaling=s), want)
    one = ops.adapted_linear(x[3], w, a, b, ids[3], scaling=s)
    assert one.shape == (136,)
    near(one.unsqueeze(0), *formula(x[3:4], w, a, b, ids[3:4], s))
    for rows in ((0,), (2, 0)):
        e = ops.adapted_linear(torch.zeros(*rows, 264, dtype=BF16, device=DEV), w, a, b,
                               torch.zeros(rows, dtype=torch.int32, device=DEV), scaling=s)
        assert e.shape == (*rows, 136)
    # no adapters are loaded
    none = ops.adapted_linear(x, w, a[:0], b[:0], ids)
    near(none, *formula(x, w, a[:0], b[:0], ids, None))
    many = inputs(300, 264, 136, 1, 16, BF16, 2)
    near(ops.adapted_linear(many[0], w, a[:0], b[:0], many[4]),
         *formula(many[0], w, a[:0], b[:0], many[4], None))
    few = ops.adapted_linear(x[:4], w, a[:0], b[:0], ids[:4], scaling=s[:0])
    near(few, *formula(x[:4], w, a[:0], b[:0], ids[:4], None))


@pytest.mark.parametrize("tokens", [7, 64, 700])
def test_graphs_and_streams(tokens):
    args = [inputs(tokens, 520, 1032, 6, 16, BF16, seed) for seed in (1, 2)]
    want = [ops.adapted_linear(*v[:5], scaling=v[5]) for v in args]
    # two calls at once
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            other = ops.adapted_linear(*args[1][:5], scaling=args[1][5])
        here = ops.adapted_linear(*args[0][:5], scaling=args[0][5])
        torch.cuda.synchronize()
        assert torch.equal(here, want[0]) and torch.equal(other, want[1])
    # one behind the other in a graph, the second on the first's result
    x, w, a, b, ids, s = args[0]
    back = inputs(tokens, 1032, 520, 6, 16, BF16, 3)
    chain = ops.adapted_linear(want[0], *back[1:5], scaling=back[5])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.adapted_linear(x, w, a, b, ids, scaling=s)
        z = ops.adapted_linear(y, *back[1:5], scaling=back[5])
    for _ in range(3):
        y.zero_()
        z.zero_()
        graph.replay()
        assert torch.equal(y, want[0]) and torch.equal(z, chain)
    # other ids in the same graph
    ids.copy_(args[1][4])
    graph.replay()
    assert torch.equal(y, ops.adapted_linear(x, w, a, b, ids, scaling=s))


def test_refusals():
    x, w, a, b, ids, s = inputs(4, 64, 32, 2, 8, BF16, 1)
    with pytest.raises(TypeError):
        ops.adapted_linear(x.float(), w, a, b, ids)
    with pytest.raises(TypeError):
        ops.adapted_linear(x, w.half(), a, b, ids)
    with pytest.raises(TypeError):
        ops.adapted_linear(x, w, a, b, ids.float())
    with pytest.raises(ValueError):
        ops.adapted_linear(x, w, a, b[:1], ids)
    with pytest.raises(ValueError):
        ops.adapted_linear(x, w, a[:, :, :-1], b, ids)
    with pytest.raises(ValueError):
        ops.adapted_linear(x, w, a, b, ids[:-1])
    with pytest.raises(ValueError):
        ops.adapted_linear(x, w, a, b, ids, scaling=s[:1])
    with pytest.raises(NotImplementedError):
        ops.adapted_linear(x[:, :60], w[:, :60], a[:, :, :60], b, ids)
    with pytest.raises(NotImplementedError):
        ops.adapted_linear(x, w, a[:, :4], b[:, :, :4], ids)
    big = torch.zeros(1, 136, 64, dtype=BF16, device=DEV)
    with pytest.raises(NotImplementedError):
        ops.adapted_linear(x, w, big, torch.zeros(1, 32, 136, dtype=BF16, device=DEV), ids)
    with pytest.raises(RuntimeError):
        ops.adapted_linear(x, w.cpu(), a, b, ids)
