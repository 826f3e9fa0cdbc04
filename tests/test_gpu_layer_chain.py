"""The operators around the expert layer in one layer, as training and serving run them: norm with the
residual, router, balance loss, routed experts, shared expert, adapted projection.  Each stage is held to its
own bounds on the inputs and upstream gradients that it met."""

from __future__ import annotations

import pytest
import torch

import test_gpu_adapted_linear as adapted
import test_gpu_balance_loss as balance
import test_gpu_rms_norm as norm
from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16 = torch.bfloat16


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_training_step(scoring):
    tokens, hidden, experts, top_k, inter = 300, 512, 64, 4, 256
    x, r, w, _, ds = norm.inputs(tokens, hidden, BF16, 1)
    g = torch.Generator(device=DEV).manual_seed(2)
    gate = torch.randn(hidden, experts, generator=g, device=DEV) / hidden ** 0.5
    w13 = (torch.randn(2 * inter, hidden, generator=g, device=DEV) / hidden ** 0.5).to(BF16)
    mask = torch.rand(tokens, generator=g, device=DEV) < 0.8
    leaves = [t.requires_grad_(True) for t in (x, r, w, gate, w13)]

    y, s = ops.rms_norm(x, w, residual=r)
    logits = y.float() @ gate
    _, ids = ops.router_topk(logits.detach(), top_k, scoring=scoring)
    loss, counts = ops.balance_loss(logits, ids, scoring=scoring, mask=mask)
    h = ops.gated_mlp(y, w13)
    for t in (y, s, logits):
        t.retain_grad()
    scale = torch.full_like(loss, 64.0)
    total = scale * loss + (h.float() * 0.01).square().sum() + (s.float() * ds.float()).sum()
    total.backward()
    assert all(t.grad is not None and bool(t.grad.isfinite().all()) for t in leaves)

    assert int(counts.sum()) == int(mask.sum()) * top_k
    want, bound = norm.formulas(s.detach(), w.detach(), y.grad, s.grad, 1e-6)
    norm.near(y.detach(), want[0], bound[0])
    norm.near(x.grad, want[1], bound[1])
    assert torch.equal(x.grad, r.grad)
    norm.near(w.grad, want[2], bound[2])
    want, bound = balance.formula(logits.detach().unsqueeze(0), ids.unsqueeze(0), mask.unsqueeze(0),
                                  scale.view(1), scoring)
    balance.near(loss.detach().view(1), want[0], bound[0])
    assert torch.equal(counts.unsqueeze(0), want[1])
    balance.near(logits.grad.unsqueeze(0), want[2], bound[1])


def layer(x, r, weights, routes, adapters, ids):
    norm_w, w13, s13, w2, s2, shared13, shared2 = weights
    y, s = ops.rms_norm(x, norm_w, residual=r)
    out = ops.fused_experts_mxfp4(y, *routes, w13, s13, w2, s2)
    h = ops.gated_mlp(y, shared13)
    return out + ops.adapted_linear(h, shared2, *adapters[:2], ids, scaling=adapters[2]), s, h


@pytest.mark.parametrize("tokens", [1, 24, 200, 1100])
def test_serving_layers(tokens):
    hidden, inter, shared, experts, top_k, count, rank = 256, 128, 264, 16, 4, 5, 16
    g = torch.Generator(device=DEV).manual_seed(tokens)

    def normal(*shape, size=1.0):
        return (size * torch.randn(*shape, generator=g, device=DEV)).to(BF16)

    w13, s13 = ops.quantize_mxfp4(normal(experts, 2 * inter, hidden, size=hidden ** -0.5))
    w2, s2 = ops.quantize_mxfp4(normal(experts, hidden, inter, size=inter ** -0.5))
    weights = (normal(hidden) + 1, w13, ops.tile_mxfp4_scales(s13), w2, ops.tile_mxfp4_scales(s2),
               normal(2 * shared, hidden, size=hidden ** -0.5),
               normal(hidden, shared, size=shared ** -0.5))
    adapters = (normal(count, rank, shared, size=shared ** -0.5),
                normal(count, hidden, rank, size=rank ** -0.5),
                0.5 + torch.rand(count, generator=g, device=DEV))
    ids = torch.randint(-1, count, (tokens,), generator=g, device=DEV)
    x, r = normal(tokens, hidden), normal(tokens, hidden)
    logits = torch.randn(tokens, 64, generator=g, device=DEV)
    tw, ti = ops.router_topk(logits, top_k)
    routes = (tw, ti % experts)

    first, s, h = layer(x, r, weights, routes, adapters, ids)
    second, s_next, _ = layer(first, s, weights, routes, adapters, ids)
    assert torch.equal(s_next, (first.float() + s.float()).to(BF16))
    got = ops.adapted_linear(h, weights[6], *adapters[:2], ids, scaling=adapters[2])
    adapted.near(got, *adapted.formula(h, weights[6], *adapters[:2], ids, adapters[2]))
    # the same layers replayed, on other inputs too
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b, _ = layer(x, r, weights, routes, adapters, ids)
        out, _, _ = layer(a, b, weights, routes, adapters, ids)
    for _ in range(2):
        graph.replay()
        assert torch.equal(out, second)
    x.copy_(normal(tokens, hidden))
    want, s, _ = layer(x, r, weights, routes, adapters, ids)
    want, _, _ = layer(want, s, weights, routes, adapters, ids)
    graph.replay()
    assert torch.equal(out, want)


def test_norm_in_8_bits_beside_the_norm():
    """The 8-bit form of a layer's norm is the norm within its codes' rounding: half a step of e4m3 (2^-4
    of a value, 2^-10 of the largest code) or of the integers (1 / 254 of a group's largest)."""
    x, r, w, _, _ = norm.inputs(300, 1000, BF16, 5)
    y, s = ops.rms_norm(x, w, residual=r)
    for dtype in (torch.float8_e4m3fn, torch.int8):
        for group in (None, 64):
            codes, scales, s8 = ops.rms_norm_8bit(x, w, residual=r, dtype=dtype, group=group)
            back = ops.dequantize_8bit(codes, scales, group=group, dtype=torch.float32).double()
            assert torch.equal(s8, s)
            wide = scales.double().repeat_interleave(group or 1000, 1)[:, :1000]
            step = (torch.maximum(back.abs() * 2.0 ** -4 * 1.07, wide * 2.0 ** -10)
                    if dtype is torch.float8_e4m3fn else wide * 0.5)
            # (y itself is rounded to bf16)
            assert bool(((back - y.double()).abs() <= step * 1.01 + y.double().abs() * 2.0 ** -8).all())
