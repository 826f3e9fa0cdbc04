"""Each of the MXFP4 expert layer's kernels at the sizes it is written for, against the formula in 64 bits:
blocks of 16, 32 and 128 routes with reductions longer than a turn of their stages, blocks that end on, before
and after a border, more routes than one align launch takes, inputs that the tensor maps need realigned.

The formula and its bounds are test_gpu_experts_mxfp4's; the result's rounding to bf16, whose values lie
2^-7 apart at 1, is counted here as the 2^-8 that it is.
"""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import _lib as L
from exfold_b200 import ops
from test_gpu_experts_mxfp4 import formula, near, routing, run, tokens_of, weights

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def not_few(tokens, top_k, experts, hidden, inter):
    """The layer for a few routes keeps the intermediate activations and nothing else."""
    size = L.lib().exf_fused_experts_mxfp4_workspace_bytes(tokens, top_k, experts, hidden, inter)
    return size > tokens * top_k * inter * 4 + 4096


def check(x, tw, ids, p13, p2):
    y = run(x, tw, ids, p13, p2)
    want, bound = formula(x, tw, ids, p13[2], p2[2])
    near(y, want, bound + 2.0 ** -9 * want.abs())
    assert torch.equal(run(x, tw, ids, p13, p2), y)
    return y


# tokens, experts, top_k, hidden, inter.  Routes an expert, masked ones counted: up to 12 take blocks of 16,
# up to 44 blocks of 32, above that the prefill kernels.
LARGE = [(24, 16, 8, 4096, 2048), (12, 32, 8, 2048, 768), (7, 12, 8, 4096, 2048),
         (60, 16, 8, 4096, 2048), (100, 24, 8, 2048, 768), (100, 16, 8, 4096, 2048)]


@pytest.mark.parametrize("tokens,experts,top_k,hidden,inter", LARGE)
def test_long_reductions(tokens, experts, top_k, hidden, inter):
    assert not_few(tokens, top_k, experts, hidden, inter)
    tw, ids = routing(tokens, experts, top_k, seed=tokens)
    p13, p2 = weights(experts, hidden, inter, seed=tokens + 1)
    x = tokens_of(tokens, hidden, seed=tokens + 2)
    check(x, tw, ids, p13, p2)
    # an expert-parallel rank: three quarters of the routes are other ranks', the last tokens are padding
    g = torch.Generator(device=DEV).manual_seed(tokens + 3)
    ids = torch.where(torch.rand(ids.shape, generator=g, device=DEV) < 0.75, -1, ids)
    ids[tokens - 2:] = -1
    y = check(x, tw, ids, p13, p2)
    assert torch.count_nonzero(y[tokens - 2:]) == 0


@pytest.mark.parametrize("experts,routes", [(16, 15), (16, 16), (16, 17), (16, 31), (16, 33), (16, 64),
                                            (16, 65), (16, 192), (2, 31), (2, 32), (2, 33), (2, 64),
                                            (2, 65), (2, 88), (1, 127), (1, 128), (1, 129), (2, 257)])
def test_block_borders(experts, routes):
    """All routes to one expert, the last: its blocks of 16, 32 or 128 end before, on or after a border."""
    hidden, inter = 2048, 1408
    assert not_few(routes, 1, experts, hidden, inter)
    p13, p2 = weights(experts, hidden, inter, seed=routes)
    x = tokens_of(routes, hidden, seed=routes + 1)
    ids = torch.full((routes, 1), experts - 1, dtype=torch.int32, device=DEV)
    tw = torch.rand(routes, 1, device=DEV) + 0.5
    check(x, tw, ids, p13, p2)


@pytest.mark.parametrize("tokens,hidden,inter", [(1025, 256, 128), (1100, 1280, 128), (1408, 512, 256)])
def test_decode_blocks_of_many_routes(tokens, hidden, inter):
    """Over 8192 routes, at most 44 an expert: blocks of 32 after an align of three launches."""
    experts, top_k = 256, 8
    tw, ids = routing(tokens, experts, top_k, seed=tokens)
    ids[5], ids[6, 3] = -1, experts
    p13, p2 = weights(experts, hidden, inter, seed=tokens + 1)
    x = tokens_of(tokens, hidden, seed=tokens + 2)
    y = check(x, tw, ids, p13, p2)
    assert torch.count_nonzero(y[5]) == 0


@pytest.mark.parametrize("tokens,experts,top_k", [(40, 16, 4), (120, 16, 4), (400, 8, 4)])
def test_unaligned_and_strided_inputs(tokens, experts, top_k):
    """Blocks of 16, 32 and 128 on weights, scales and activations at odd addresses."""
    hidden, inter = 1024, 512
    assert not_few(tokens, top_k, experts, hidden, inter)
    tw, ids = routing(tokens, experts, top_k, seed=10)
    p13, p2 = weights(experts, hidden, inter, seed=11)
    x = tokens_of(tokens, hidden, seed=12)
    want = check(x, tw, ids, p13, p2)
    wide = torch.zeros(tokens, hidden + 5, dtype=torch.bfloat16, device=DEV)
    wide[:, 5:] = x

    def shifted(t, n):
        flat = torch.empty(t.numel() + n, dtype=t.dtype, device=DEV)
        flat[n:] = t.reshape(-1)
        return flat[n:].view(t.shape)

    for shifts in ((1, 3, 16, 8), (16, 8, 1, 3), (32, 16, 16, 16)):
        got = ops.fused_experts_mxfp4(
            wide[:, 5:], tw.double(), ids.long(), shifted(p13[0], shifts[0]),
            shifted(ops.tile_mxfp4_scales(p13[1]), shifts[1]), shifted(p2[0], shifts[2]),
            shifted(ops.tile_mxfp4_scales(p2[1]), shifts[3]))
        assert torch.equal(got, want)


@pytest.mark.parametrize("tokens,top_k", [(48, 8), (160, 8), (700, 8)])
def test_routes_on_a_few_experts(tokens, top_k):
    """Routes that a fold or a decode budget sent to 9 of 32 experts, some twice in a token."""
    experts, hidden, inter = 32, 1024, 256
    assert not_few(tokens, top_k, experts, hidden, inter)
    g = torch.Generator(device=DEV).manual_seed(tokens)
    some = torch.randperm(experts, generator=g, device=DEV)[:9].int()
    ids = some[torch.randint(0, 9, (tokens, top_k), generator=g, device=DEV)]
    tw = torch.rand(tokens, top_k, generator=g, device=DEV)
    p13, p2 = weights(experts, hidden, inter, seed=tokens + 1)
    check(tokens_of(tokens, hidden, seed=tokens + 2), tw, ids, p13, p2)


@pytest.mark.parametrize("tokens", [2, 40, 300, 800])  # a few routes, blocks of 16, 32, 128
def test_calls_that_read_what_the_one_before_wrote(tokens):
    """Router, experts, gated block and experts again with nothing between the launches, eagerly and by
    graph, against the same calls with the device idle before each: a kernel is resident before its
    predecessor has finished, and reads its results only after."""
    hidden, inter, experts, top_k = 512, 256, 64, 4
    p13, p2 = weights(experts, hidden, inter, seed=tokens)
    t13, t2 = ops.tile_mxfp4_scales(p13[1]), ops.tile_mxfp4_scales(p2[1])
    g = torch.Generator(device=DEV).manual_seed(tokens + 1)
    w = (torch.randn(2 * hidden, hidden, generator=g, device=DEV) / hidden ** 0.5).bfloat16()
    logits = torch.randn(tokens, experts, generator=g, device=DEV)
    x = tokens_of(tokens, hidden, seed=tokens + 2)

    def chain(between):
        outs = []
        y = x
        for k in range(3):
            tw, ids = ops.router_topk(logits, top_k, renormalize=k > 0)
            between()
            y = ops.fused_experts_mxfp4(y, tw, ids, p13[0], t13, p2[0], t2)
            between()
            outs.append(y)
            y = ops.gated_mlp(y, w)
            between()
            outs.append(y)
        return outs

    want = chain(torch.cuda.synchronize)
    assert torch.count_nonzero(want[0]) > 0
    for _ in range(5):
        for a, b in zip(chain(lambda: None), want):
            assert torch.equal(a.nan_to_num(), b.nan_to_num())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(lambda: None)
    for _ in range(5):
        graph.replay()
    for a, b in zip(got, want):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
