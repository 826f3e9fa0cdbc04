"""The expert layer with MXFP4 weights against its formula in 64 bits.

Bounds, element by element (u = 2^-8 / 2 for the bf16 result; t = 2 k 2^-23 for a sum of k terms in two
fp32 chains):
  activations enter within e_x = 2^-22 max|x| of their block of 32;
  |dG| <= (e_x + t |x|) |W|^T =: a (the same for U); the logistic function within r = 2^-19;
  |dh| <= 1.13 a |U| + (|act| + 1.13 a) a + 2 r |h|, then its two-term form: 2^-9 |h| plus
  2^-22 of the largest |h| of its block of 32;
  |dy| <= sum_j w_j (|dh| + t |h|) |W2|^T + 9 * 2^-24 sum_j |w_j o_j| + u |y|, and 2^-14 of the largest
  |w_j o_j| of its 32 columns where route outputs are held in 16 bits (multiples of a power of two u
  with that largest in [2^13 u, 2^14 u), so within u / 2; never below u = 2^-126).
"""

from __future__ import annotations

import math

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def weights(experts, hidden, inter, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def make(rows, cols):
        w = torch.randn(experts, rows, cols, generator=g, device=DEV) / math.sqrt(cols)
        size = torch.exp2(4 * torch.rand(experts, rows, 1, generator=g, device=DEV) - 2)
        codes, scales = ops.quantize_mxfp4(w * size)
        return codes, scales, ops.dequantize_mxfp4(codes, scales, dtype=torch.float32).double()

    return make(2 * inter, hidden), make(hidden, inter)


def tokens_of(tokens, hidden, seed):
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    x = torch.randn(tokens, hidden, generator=g, device=DEV)
    x = x * torch.exp2(3 * torch.rand(tokens, hidden, generator=g, device=DEV))
    return x.bfloat16()


def routing(tokens, experts, top_k, seed):
    g = torch.Generator(device=DEV).manual_seed(seed + 2)
    w, ids = torch.softmax(torch.randn(tokens, experts, generator=g, device=DEV), -1).topk(top_k)
    return w.contiguous(), ids.int().contiguous()


def block_max(v):
    return v.abs().reshape(v.shape[0], -1, 32).amax(-1).repeat_interleave(32, -1)


def formula(x, tw, ids, w13, w2):
    x, tw = x.double(), tw.double()
    hidden, inter = x.shape[1], w13.shape[1] // 2
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    t1, t2, r = 2 * hidden * 2.0 ** -23, 2 * inter * 2.0 ** -23, 2.0 ** -19
    ex = 2.0 ** -22 * block_max(x) + t1 * x.abs()
    for e in range(w13.shape[0]):
        at, slot = torch.nonzero(ids == e, as_tuple=True)
        if at.numel() == 0:
            continue
        g, u = (x[at] @ w13[e].t()).chunk(2, 1)
        ag, au = (ex[at] @ w13[e].abs().t()).chunk(2, 1)
        act = g * torch.sigmoid(g)
        h = act * u
        ea = 1.13 * ag + 2 * r * act.abs()
        eh = ea * (u.abs() + au) + act.abs() * au
        eh = eh * (1 + 2.0 ** -9) + 2.0 ** -9 * h.abs() + 2.0 ** -22 * block_max(h.abs() + eh)
        o = h @ w2[e].t()
        eo = (eh + t2 * (h.abs() + eh)) @ w2[e].abs().t()
        w = tw[at, slot].unsqueeze(1)
        y.index_add_(0, at, w * o)
        bound.index_add_(0, at, w.abs() * (eo + 9 * 2.0 ** -24 * (o.abs() + eo)))
        if ids.numel() > 44 * w13.shape[0]:
            bound.index_add_(0, at, 2.0 ** -14 * block_max(w.abs() * (o.abs() + eo)) + 2.0 ** -127)
    return y, bound * (1 + 2.0 ** -8) + 2.0 ** -9 * y.abs() + 2.0 ** -134


def run(x, tw, ids, packed13, packed2):
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    y = ops.fused_experts_mxfp4(x, tw, ids, packed13[0], ops.tile_mxfp4_scales(packed13[1]),
                                packed2[0], ops.tile_mxfp4_scales(packed2[1]), status=status)
    assert int(status) == 0, "a pipeline wait timed out"
    return y


def near(y, want, bound):
    off = (y.double() - want).abs()
    assert bool((off <= bound).all()), (
        f"off by {(off / bound.clamp(min=1e-300)).max().item():.3g} bounds")


CASES = [  # tokens, experts, top_k, hidden, inter: routes per expert from below 1 to hundreds
    (1, 8, 2, 256, 128), (1, 128, 8, 2048, 768), (3, 4, 1, 512, 256), (7, 16, 8, 768, 384),
    (16, 8, 8, 256, 128), (17, 1, 1, 256, 128), (33, 1, 1, 512, 128), (64, 1, 1, 256, 256),
    (65, 1, 1, 256, 128), (100, 8, 3, 1024, 640), (256, 128, 8, 2048, 768), (300, 16, 4, 512, 256),
    (500, 8, 2, 4096, 256), (1000, 8, 4, 256, 1152), (2500, 12, 5, 512, 384),
    (1100, 3, 8, 512, 128)]


@pytest.mark.parametrize("tokens,experts,top_k,hidden,inter", CASES)
def test_against_formula(tokens, experts, top_k, hidden, inter):
    if top_k > experts:  # an expert named several times by a token counts as often
        ids = torch.arange(top_k, dtype=torch.int32, device=DEV).remainder(experts)
        ids = ids.expand(tokens, top_k).contiguous()
        tw = torch.rand(tokens, top_k, device=DEV)
    else:
        tw, ids = routing(tokens, experts, top_k, seed=tokens)
    p13, p2 = weights(experts, hidden, inter, seed=tokens + experts)
    x = tokens_of(tokens, hidden, seed=tokens)
    y = run(x, tw, ids, p13, p2)
    near(y, *formula(x, tw, ids, p13[2], p2[2]))
    assert torch.equal(run(x, tw, ids, p13, p2), y)


def test_masked_routes_and_tokens():
    """Ids of -1 and >= experts contribute nothing, whatever their weight; a token without a valid
    route gives 0, and a padded batch's last rows too."""
    for tokens, experts in ((20, 16), (40, 16), (900, 8)):
        tw, ids = routing(tokens, experts, 4, seed=1)
        p13, p2 = weights(experts, 512, 256, seed=2)
        x = tokens_of(tokens, 512, seed=3)
        ids[0], ids[1, 1], ids[2, 1], ids[3] = -1, experts, ids[2, 0], 5
        ids[4] = torch.tensor([-1, experts + 7, 3, -(1 << 31)], dtype=torch.int32)
        ids[tokens - 7:] = -1
        tw[0], tw[1, 1] = math.nan, math.inf
        x[tokens - 3:] = math.nan
        y = run(x, tw, ids, p13, p2)
        clean, zero = x.clone(), tw.clone()
        clean[tokens - 3:], zero[0], zero[1, 1] = 0.0, 0.0, 0.0
        near(y, *formula(clean, zero, ids, p13[2], p2[2]))
        assert torch.count_nonzero(y[0]) == 0 and torch.count_nonzero(y[tokens - 7:]) == 0
    y = run(x, tw, torch.full_like(ids, -1), p13, p2)
    assert torch.count_nonzero(y) == 0


def test_prefill_values_far_apart():
    """The 16-bit route outputs: expert outputs from 2^-100 to 2^100, empty and NaN ones."""
    tw, ids = routing(700, 4, 2, seed=30)
    p13, p2 = weights(4, 256, 128, seed=31)
    x = tokens_of(700, 256, seed=32)
    size = torch.exp2(torch.arange(700, device=DEV) % 100 - 50.0).unsqueeze(1)
    x = (x.float() * size).bfloat16()
    x[5] = 0.0
    tw[6] = 0.0
    y = run(x, tw, ids, p13, p2)
    near(y, *formula(x, tw, ids, p13[2], p2[2]))
    tw[7, 0], tw[8, 1] = math.nan, math.inf
    got = run(x, tw, ids, p13, p2)
    keep = [i for i in range(700) if i not in (7, 8)]
    assert torch.equal(got[keep], y[keep])
    assert not bool(torch.isfinite(got[7:9]).any())


@pytest.mark.parametrize("tokens,experts", [(20, 4), (160, 8), (400, 4)])
@pytest.mark.parametrize("size", [3.0, 2.0 ** 20, 2.0 ** 60])
def test_tiny_outputs_and_large_weights(tokens, experts, size):
    """Expert outputs about 2^-115 with routing weights of 3 and more (a two-term value is held to
    2^-137: half a step of its second term's smallest)."""
    tw, ids = routing(tokens, experts, 2, seed=33)
    p13, p2 = weights(experts, 256, 128, seed=34)
    x = (tokens_of(tokens, 256, seed=35).float() * 2.0 ** -60).bfloat16()
    want, bound = formula(x, tw * size, ids, p13[2], p2[2])
    floor = 2.0 ** -137 * size * p2[2].abs().sum(-1).amax()
    near(run(x, tw * size, ids, p13, p2), want, bound + floor)


@pytest.mark.parametrize("tokens", [48, 160, 400])  # the layer for a few routes, decode, prefill
def test_values_far_apart_and_not_finite(tokens):
    """Blocks of zeros, of the smallest and of large values; a token with an infinity or NaN gives
    NaN and leaves the others as they are."""
    tw, ids = routing(tokens, 8, 2, seed=4)
    p13, p2 = weights(8, 256, 128, seed=5)
    x = tokens_of(tokens, 256, seed=6)
    x[0] = 0.0
    x[1, 32:64] = 0.0
    x[2] = 2.0 ** -133                      # bf16's smallest subnormal
    x[3, :128] *= 2.0 ** -100
    x[4, :32] *= 2.0 ** 20
    x[5, 0] = 2.0 ** 15                     # one value far above its block
    x[6] *= 2.0 ** 10
    y = run(x, tw, ids, p13, p2)
    near(y, *formula(x, tw, ids, p13[2], p2[2]))
    bad = x.clone()
    bad[7, 9], bad[8, 200], bad[9, 3] = math.inf, math.nan, -math.inf
    got = run(bad, tw, ids, p13, p2)
    keep = [i for i in range(tokens) if i not in (7, 8, 9)]
    assert torch.equal(got[keep], y[keep])
    assert bool(torch.isnan(got[7:10]).all())


@pytest.mark.parametrize("tokens,experts", [(30, 2), (150, 16), (150, 2)])
def test_scales_at_their_limits(tokens, experts):
    """Every code against scales from 2^-127 up, and the NaN scale of one weight row."""
    g = torch.Generator(device=DEV).manual_seed(8)
    w13 = torch.randint(0, 256, (experts, 256, 128), generator=g, device=DEV).to(torch.uint8)
    w2 = torch.randint(0, 256, (experts, 256, 64), generator=g, device=DEV).to(torch.uint8)
    s13 = torch.randint(110, 124, (experts, 256, 8), generator=g, device=DEV).to(torch.uint8)
    s2 = torch.randint(110, 124, (experts, 256, 4), generator=g, device=DEV).to(torch.uint8)
    s13[0, :, 3], s2[1, 7] = 0, 0
    s2[0, 9, 2] = 255
    v13 = ops.dequantize_mxfp4(w13, s13, dtype=torch.float32).double()
    v2 = ops.dequantize_mxfp4(w2, s2, dtype=torch.float32).double()
    x = tokens_of(tokens, 256, seed=9)
    ids = torch.arange(tokens, device=DEV).remainder(experts).int().unsqueeze(1)
    tw = torch.ones(tokens, 1, device=DEV)
    y = run(x, tw, ids, (w13, s13), (w2, s2))
    assert bool(torch.isnan(y[::experts, 9]).all())
    y[::experts, 9] = 0.0
    v2[0, 9] = 0.0
    near(y, *formula(x, tw, ids, v13, v2))


def test_unaligned_and_strided_inputs():
    tw, ids = routing(20, 8, 4, seed=10)
    p13, p2 = weights(8, 256, 128, seed=11)
    x = tokens_of(20, 256, seed=12)
    wide = torch.zeros(20, 261, dtype=torch.bfloat16, device=DEV)
    wide[:, 5:] = x

    def shifted(t, n):
        flat = torch.empty(t.numel() + n, dtype=t.dtype, device=DEV)
        flat[n:] = t.reshape(-1)
        return flat[n:].view(t.shape)

    far = ids.long()
    far[3, 1] += 1 << 32  # out of range, although its low 32 bits are an expert
    masked = ids.clone()
    masked[3, 1] = -1
    want = run(x, tw, masked, p13, p2)
    got = ops.fused_experts_mxfp4(
        wide[:, 5:], tw.double(), far, shifted(p13[0], 1),
        shifted(ops.tile_mxfp4_scales(p13[1]), 3), shifted(p2[0], 16),
        shifted(ops.tile_mxfp4_scales(p2[1]), 8))
    assert torch.equal(got, want)


def test_streams_and_graphs():
    """Two graphs captured over the same inputs and an eager call on another stream give the same
    values; a replay follows its inputs, routes included."""
    tw, ids = routing(120, 16, 4, seed=13)
    p13, p2 = weights(16, 512, 256, seed=14)
    x = tokens_of(120, 512, seed=15)
    want = run(x, tw, ids, p13, p2)
    t13, t2 = ops.tile_mxfp4_scales(p13[1]), ops.tile_mxfp4_scales(p2[1])

    def call():
        return ops.fused_experts_mxfp4(x, tw, ids, p13[0], t13, p2[0], t2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(call())
    x.copy_(tokens_of(120, 512, seed=16))
    ids.copy_(routing(120, 16, 4, seed=17)[1])
    ids[100:] = -1
    want = call()
    for graph in graphs:
        graph.replay()
    for out in outs:
        assert torch.equal(out, want)


@pytest.mark.parametrize("tokens,experts", [(20, 4), (160, 8), (400, 4)])
def test_results_not_finite_stay_in_their_columns(tokens, experts):
    """Columns of the down projection whose scale is NaN, and ones whose route outputs overflow: NaN or
    an infinity there, everywhere else what the call gives without them."""
    hidden, inter = 512, 128
    tw, ids = routing(tokens, experts, 2, seed=70)
    p13, p2 = weights(experts, hidden, inter, seed=71)
    x = tokens_of(tokens, hidden, seed=72)
    want, bound = formula(x, tw, ids, p13[2], p2[2])
    near(run(x, tw, ids, p13, p2), want, bound)
    codes, scales = p2[0].clone(), p2[1].clone()
    scales[0, 9] = 255
    scales[:, 300] = 254                    # sums near 2^127 * 6 * |h|: beyond fp32
    codes[:, 300] = 0x77                    # 6
    y = run(x, tw, ids, p13, (codes, scales))
    first = (ids == 0).any(-1)
    assert bool(torch.isnan(y[first, 9]).all())
    assert bool(torch.isinf(y[:, 300]).any()) and not bool(torch.isfinite(y[:, 300]).all())
    others = torch.ones(hidden, dtype=torch.bool, device=DEV)
    others[[9, 300]] = False
    near(y[:, others], want[:, others], bound[:, others])
    rest = ~first
    near(y[rest, 9], want[rest, 9], bound[rest, 9])


@pytest.mark.parametrize("top_k", range(1, 9))
def test_few_routes(top_k):
    """One to 16 tokens, every number of routes a token, lengths of one to eleven groups of 128."""
    for tokens, hidden, inter in ((1, 1408, 1408), (3, 256, 896), (16, 512, 128)):
        hidden = hidden // 256 * 256
        tw, ids = routing(tokens, 12, top_k, seed=50 + top_k)
        if tokens == 3:
            ids[1, 0], ids[2, top_k - 1] = -1, 12
        p13, p2 = weights(12, hidden, inter, seed=51 + top_k)
        x = tokens_of(tokens, hidden, seed=52 + top_k)
        y = run(x, tw, ids, p13, p2)
        near(y, *formula(x, tw, ids, p13[2], p2[2]))


def test_few_routes_by_graph_between_other_calls():
    """Calls of one token in a row on a stream, each reading what the one before it wrote, in a graph."""
    p13, p2 = weights(8, 256, 128, seed=60)
    tw, ids = routing(1, 8, 4, seed=61)
    x = tokens_of(1, 256, seed=62)
    t13, t2 = ops.tile_mxfp4_scales(p13[1]), ops.tile_mxfp4_scales(p2[1])

    def chain():
        y = x
        for _ in range(12):
            y = ops.fused_experts_mxfp4(y, tw, ids, p13[0], t13, p2[0], t2)
            y = torch.tanh(y) + x
        return y

    want = x
    for _ in range(12):
        want = ops.fused_experts_mxfp4(want, tw, ids, p13[0], t13, p2[0], t2)
        torch.cuda.synchronize()
        want = torch.tanh(want) + x
    assert torch.equal(chain(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for _ in range(3):
        graph.replay()
    assert torch.equal(got, want)


def test_no_tokens():
    p13, p2 = weights(8, 256, 128, seed=18)
    x = torch.empty(0, 256, dtype=torch.bfloat16, device=DEV)
    y = run(x, torch.empty(0, 4, device=DEV), torch.empty(0, 4, dtype=torch.int32, device=DEV),
            p13, p2)
    assert y.shape == (0, 256)


@pytest.mark.parametrize("tokens", [1, 6, 300])
def test_moe_block_with_shared_expert(tokens):
    """A whole block as a model runs it: router, routed MXFP4 experts and the shared expert (the gated
    block, then its down projection), one token, a decode batch and a prefill batch."""
    hidden, inter, experts, top_k = 512, 256, 64, 8
    g = torch.Generator(device=DEV).manual_seed(19)
    gate = torch.randn(experts, hidden, generator=g, device=DEV) / math.sqrt(hidden)
    p13, p2 = weights(experts, hidden, inter, seed=20)
    shared13 = (torch.randn(2 * inter, hidden, generator=g, device=DEV) / math.sqrt(hidden)).bfloat16()
    shared2 = (torch.randn(hidden, inter, generator=g, device=DEV) / math.sqrt(inter)).bfloat16()
    x = tokens_of(tokens, hidden, seed=21)
    tw, ids = ops.router_topk(x.float() @ gate.t(), top_k)
    routed = run(x, tw, ids, p13, p2)
    y = routed + ops.gated_mlp(x, shared13) @ shared2.t()
    want, bound = formula(x, tw, ids, p13[2], p2[2])
    gt, up = (x.double() @ shared13.double().t()).chunk(2, 1)
    h = gt * torch.sigmoid(gt) * up
    s = h @ shared2.double().t()
    # the shared expert: h within 3 * 2^-9 of itself and of the sums' error, one rounding of each
    # bf16 result (h, s, the sum)
    t = 2 * hidden * 2.0 ** -23 * (x.double().abs() @ shared13.double().abs().t())
    eg, eu = t.chunk(2, 1)
    eh = 1.13 * eg * (up.abs() + eu) + (gt * torch.sigmoid(gt)).abs() * eu + 2.0 ** -8 * h.abs()
    es = (eh + inter * 2.0 ** -23 * (h.abs() + eh)) @ shared2.double().abs().t()
    es = es * (1 + 2.0 ** -8) + 2.0 ** -9 * s.abs()
    near(y, want + s, (bound + es) * (1 + 2.0 ** -8) + 2.0 ** -9 * (want + s).abs())


def test_calls_at_once_on_three_streams():
    """A decode and a prefill call in flight together with one of a few routes, many times."""
    sets = []
    for k, (tokens, experts, top_k) in enumerate([(60, 16, 4), (900, 8, 4), (2, 8, 4)]):
        tw, ids = routing(tokens, experts, top_k, seed=40 + k)
        p13, p2 = weights(experts, 512, 384, seed=42 + k)
        x = tokens_of(tokens, 512, seed=44 + k)
        t13, t2 = ops.tile_mxfp4_scales(p13[1]), ops.tile_mxfp4_scales(p2[1])

        def call(x=x, tw=tw, ids=ids, w13=p13[0], t13=t13, w2=p2[0], t2=t2):
            return ops.fused_experts_mxfp4(x, tw, ids, w13, t13, w2, t2)

        sets.append((call, call(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for call, _, stream in sets:
            with torch.cuda.stream(stream):
                got.append(call())
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, sets[i % 3][1])
