"""The MXFP4 expert layer with ids of every integer type against the same ids as int32."""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("tokens", [2, 120, 900])  # a few routes, decode and prefill
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int64])
def test_ids_of_every_integer_type(dtype, tokens):
    hidden, inter, experts, top_k = 256, 128, 16, 4
    g = torch.Generator(device=DEV).manual_seed(tokens)
    w13, s13 = ops.quantize_mxfp4(torch.randn(experts, 2 * inter, hidden, generator=g, device=DEV))
    w2, s2 = ops.quantize_mxfp4(torch.randn(experts, hidden, inter, generator=g, device=DEV))
    s13, s2 = ops.tile_mxfp4_scales(s13), ops.tile_mxfp4_scales(s2)
    x = torch.randn(tokens, hidden, generator=g, device=DEV).bfloat16()
    tw, ids = torch.softmax(torch.randn(tokens, experts, generator=g, device=DEV), -1).topk(top_k)
    ids[1, 2], ids[1, 3] = 100, 127  # no expert of this layer
    want = ops.fused_experts_mxfp4(x, tw, ids.int(), w13, s13, w2, s2)
    assert torch.count_nonzero(want) > want.numel() // 2
    got = ops.fused_experts_mxfp4(x, tw, ids.to(dtype), w13, s13, w2, s2)
    assert torch.equal(got, want)
    with pytest.raises(TypeError):
        ops.fused_experts_mxfp4(x, tw, ids.float(), w13, s13, w2, s2)
