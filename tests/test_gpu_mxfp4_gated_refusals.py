"""Refusals of the Python front end that need CUDA tensors: types and shapes that do not fit."""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_quantize():
    with pytest.raises(TypeError):
        ops.quantize_mxfp4(torch.zeros(4, 32, dtype=torch.float64, device=DEV))
    with pytest.raises(TypeError):
        ops.quantize_mxfp4(torch.zeros(4, 32, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        ops.quantize_mxfp4(torch.zeros((), device=DEV))
    codes = torch.zeros(4, 32, dtype=torch.uint8, device=DEV)
    scales = torch.zeros(4, 2, dtype=torch.uint8, device=DEV)
    for bad in ((codes[:, :31], scales, None), (codes, scales[:3], None), (codes, scales, 65),
                (codes, scales, 32), (codes, scales, -1)):
        with pytest.raises(ValueError):
            ops.dequantize_mxfp4(*bad)
    with pytest.raises(TypeError):
        ops.dequantize_mxfp4(codes, scales, dtype=torch.float64)
    with pytest.raises(TypeError):
        ops.dequantize_mxfp4(codes.int(), scales)
    assert ops.dequantize_mxfp4(codes, scales, 33).shape == (4, 33)


def test_gated():
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(32, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(TypeError):
        ops.gated_mlp(x.float(), w.float())
    with pytest.raises(TypeError):
        ops.gated_mlp(x, w.half())
    with pytest.raises(ValueError):
        ops.gated_mlp(x, w, activation="relu")
    for bad in (w[:31], w[:, :32], w[0], w[:0]):
        with pytest.raises(ValueError):
            ops.gated_mlp(x, bad)
    with pytest.raises(ValueError):
        ops.gated_mlp(x[:, :0], w[:, :0])
    with pytest.raises(NotImplementedError):
        ops.gated_mlp(x[:, :60], w[:, :60])
    with pytest.raises(NotImplementedError):
        ops.gated_mlp(x, w[:24 - 4])
    for status in (torch.zeros(1, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)):
        with pytest.raises(TypeError):
            ops.gated_mlp(x, w, status=status)


def test_experts():
    e, h, i = 4, 256, 128

    def make(dtype=torch.bfloat16, tokens=3, hidden=h, inter=i, k=2):
        u8 = {"dtype": torch.uint8, "device": DEV}
        return {"x": torch.zeros(tokens, hidden, dtype=dtype, device=DEV),
                "topk_w": torch.zeros(tokens, k, device=DEV),
                "topk_ids": torch.zeros(tokens, k, dtype=torch.int32, device=DEV),
                "w13": torch.zeros(e, 2 * inter, hidden // 2, **u8),
                "s13": torch.zeros(e, 2 * inter // 128, hidden // 128, 512, **u8),
                "w2": torch.zeros(e, hidden, inter // 2, **u8),
                "s2": torch.zeros(e, hidden // 128, inter // 128, 512, **u8)}

    ops.fused_experts_mxfp4(**make())
    with pytest.raises(TypeError):
        ops.fused_experts_mxfp4(**make(dtype=torch.float16))
    for bad in ({"hidden": 128}, {"inter": 192}, {"k": 9}):
        with pytest.raises(NotImplementedError):
            ops.fused_experts_mxfp4(**make(**bad))
    for name in ("topk_w", "w13", "s13", "w2", "s2"):
        args = make()
        args[name] = args[name][1:]
        with pytest.raises((ValueError, NotImplementedError)):
            ops.fused_experts_mxfp4(**args)
        args = make()
        args[name] = args[name].float() if args[name].dtype == torch.uint8 else args[name][:, :1]
        with pytest.raises((TypeError, ValueError)):
            ops.fused_experts_mxfp4(**args)
