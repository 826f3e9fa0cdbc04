"""The projection with adapters where a block computes many tiles: an adapter's infinities and NaN reach all of
its own tokens' features and nothing else, in every tile.

With B broken in the columns that the test names, y there is z's product with an infinity (its sign, or a NaN
where z is 0 or B is a NaN); elsewhere the result is the whole adapter's, to the bit.
"""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16 = torch.bfloat16, torch.float16


def inputs(tokens, inner, outer, adapters, rank, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return (torch.randn(*shape, generator=g, device=DEV) * shape[-1] ** -0.5).to(dtype)

    return (normal(tokens, inner), normal(outer, inner), normal(adapters, rank, inner),
            normal(adapters, outer, rank))


def adapters_of(tokens, pattern):
    """Ids by tiles of 128 tokens; pattern: the adapter of each tile in turn, -1 for none."""
    tile = torch.arange(tokens, device=DEV) // 128
    return torch.tensor(pattern, device=DEV, dtype=torch.int32)[tile % len(pattern)]


PATTERNS = [[0], [0, -1], [0, -1, -1, 0, 0, -1], [0, 1], [0, 0, 1, -1, 1], [-1] * 9 + [0]]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,inner,outer,rank", [
    (8192, 2048, 2048, 16), (8192, 2048, 4096, 8), (8192, 256, 4096, 16), (8192, 1024, 2048, 64),
    (4200, 520, 4104, 24), (1100, 264, 16392, 16), (1000, 512, 16384, 40)])
def test_broken_columns_in_every_tile(tokens, inner, outer, rank, dtype):
    x, w, a, b = inputs(tokens, inner, outer, 2, rank, dtype, tokens + rank)
    broken = b.clone()
    for at, value in ((5, "inf"), (outer // 2 + 3, "nan"), (outer - 1, "-inf")):
        broken[0, at, (3 * at) % rank] = float(value)
    good = torch.ones(outer, dtype=torch.bool, device=DEV)
    good[[5, outer // 2 + 3, outer - 1]] = False
    for pattern in PATTERNS:
        ids = adapters_of(tokens, pattern)
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        want = ops.adapted_linear(x, w, a, b, ids)
        y = ops.adapted_linear(x, w, a, broken, ids, status=status)
        assert int(status) == 0
        own = ids == 0
        assert torch.equal(y[~own], want[~own])
        assert torch.equal(y[:, good], want[:, good])
        assert bool(y[own][:, outer // 2 + 3].isnan().all())
        for at, sign in ((5, 1.0), (outer - 1, -1.0)):
            got = y[own][:, at].double()
            assert bool((got.isinf() | got.isnan()).all())
            # (where z is far enough from 0 for its sign: its rows' products are off by 2^-10 at most)
            z = sign * (x[own].double() @ a[0, (3 * at) % rank].double())
            sure = z.abs() > 2.0 ** -10
            assert torch.equal(got[sure], z[sure] * float("inf"))


@pytest.mark.parametrize("value", ["nan", "inf"])
@pytest.mark.parametrize("rank", [8, 16, 64])
def test_wholly_broken_adapter(rank, value):
    """All of B: none of the adapter's tokens has a finite feature, whichever tile they lie in."""
    tokens, inner, outer = 8192, 2048, 4096
    x, w, a, b = inputs(tokens, inner, outer, 2, rank, BF16, rank)
    broken = b.clone()
    broken[0] = float(value)
    for pattern in PATTERNS:
        ids = adapters_of(tokens, pattern)
        own = ids == 0
        y = ops.adapted_linear(x, w, a, broken, ids)
        assert not bool(y[own].isfinite().any())
        assert torch.equal(y[~own], ops.adapted_linear(x, w, a, b, ids)[~own])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,inner,outer,rank", [
    (1100, 264, 520, 16), (2500, 1024, 2048, 24), (8192, 520, 2056, 64), (4200, 256, 264, 128)])
def test_broken_rows_of_a_and_x(tokens, inner, outer, rank, dtype):
    """A NaN or an infinity of an adapter's A reaches its own tokens alone; one of a token's x that token."""
    x, w, a, b = inputs(tokens, inner, outer, 3, rank, dtype, tokens)
    for pattern in ([0, 1, 2], [1, -1, 0, 2, 2]):
        ids = adapters_of(tokens, pattern)
        ids[7::10] = 1
        want = ops.adapted_linear(x, w, a, b, ids)
        for value in ("nan", "inf"):
            broken = a.clone()
            broken[1, rank - 1, inner - 3] = float(value)
            broken[1, 0, 2] = float(value)
            y = ops.adapted_linear(x, w, broken, b, ids)
            assert not bool(y[ids == 1].isfinite().any())
            assert torch.equal(y[ids != 1], want[ids != 1])
            z = x.clone()
            z[tokens // 2, 5] = float(value)
            y = ops.adapted_linear(z, w, a, b, ids)
            assert not bool(y[tokens // 2].isfinite().any())
            others = torch.arange(tokens, device=DEV) != tokens // 2
            assert torch.equal(y[others], want[others])


@pytest.mark.parametrize("tokens", [129, 1100, 2500])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_graphs_and_streams(tokens, dtype):
    args = [inputs(tokens, 520, 4104, 6, 40, dtype, seed) for seed in (1, 2)]
    ids = [adapters_of(tokens, p) for p in ([0, 5, -1, 2], [3, 3, 1])]
    want = [ops.adapted_linear(*v, i) for v, i in zip(args, ids)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(10):  # two calls at once
        with torch.cuda.stream(side):
            other = ops.adapted_linear(*args[1], ids[1])
        here = ops.adapted_linear(*args[0], ids[0])
        torch.cuda.synchronize()
        assert torch.equal(here, want[0]) and torch.equal(other, want[1])
    graph = torch.cuda.CUDAGraph()
    who = ids[0].clone()
    with torch.cuda.graph(graph):
        y = ops.adapted_linear(*args[0], who)
        z = ops.adapted_linear(*args[1], who)
    for i in (ids[0], ids[1], ids[0]):
        who.copy_(i)
        y.zero_()
        z.zero_()
        graph.replay()
        assert torch.equal(y, ops.adapted_linear(*args[0], i))
        assert torch.equal(z, ops.adapted_linear(*args[1], i))
