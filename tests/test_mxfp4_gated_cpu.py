"""Refusals of the MXFP4 and gated feed-forward entry points: bad arguments come back as errors
before anything touches the device."""

from __future__ import annotations

import ctypes

import pytest
import torch

from exfold_b200 import _lib as L
from exfold_b200 import ops

FAKE = ctypes.c_void_p(64)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(72)


def call(name, *args):
    rc = getattr(L.lib(), name)(*args)
    return rc, L.lib().exf_last_error().decode()


def refused(got, code, word):
    rc, message = got
    assert rc == code and word in message, (rc, message)


def test_quantize_refusals():
    q = "exf_mxfp4_quantize"
    refused(call(q, FAKE, 3, 4, 32, 32, FAKE, FAKE, None), L.EXF_ERR_INVALID, "dtype")
    refused(call(q, FAKE, 0, -1, 32, 32, FAKE, FAKE, None), L.EXF_ERR_INVALID, "shape")
    refused(call(q, FAKE, 0, 4, 32, 31, FAKE, FAKE, None), L.EXF_ERR_INVALID, "row_stride")
    refused(call(q, FAKE, 0, 1 << 39, 1 << 39, 1 << 39, FAKE, FAKE, None), L.EXF_ERR_INVALID, "shape")
    refused(call(q, None, 0, 4, 32, 32, FAKE, FAKE, None), L.EXF_ERR_INVALID, "null")
    refused(call(q, FAKE, 0, 4, 32, 32, ODD, FAKE, None), L.EXF_ERR_INVALID, "aligned")
    refused(call(q, ctypes.c_void_p(66), 0, 4, 32, 32, FAKE, FAKE, None), L.EXF_ERR_INVALID,
            "aligned")
    assert call(q, None, 0, 0, 32, 32, None, None, None)[0] == 0
    d = "exf_mxfp4_dequantize"
    refused(call(d, FAKE, FAKE, 4, 32, FAKE, 9, None), L.EXF_ERR_INVALID, "dtype")
    refused(call(d, ODD, FAKE, 4, 32, FAKE, 0, None), L.EXF_ERR_INVALID, "aligned")
    refused(call(d, FAKE, FAKE, 4, 32, None, 0, None), L.EXF_ERR_INVALID, "null")
    assert call(d, None, None, 4, 0, None, 0, None)[0] == 0


def experts(tokens=4, top_k=8, w13=FAKE, e=16, hidden=256, inter=128, ws=FAKE, size=1 << 40):
    return call("exf_fused_experts_mxfp4", FAKE, FAKE, FAKE, tokens, top_k, w13, FAKE, FAKE, FAKE, e,
                hidden, inter, FAKE, ws, size, None, None)


def test_experts_refusals():
    refused(experts(top_k=9), L.EXF_ERR_UNSUPPORTED, "top_k")
    refused(experts(top_k=0), L.EXF_ERR_INVALID, "shape")
    refused(experts(e=513), L.EXF_ERR_UNSUPPORTED, "experts")
    refused(experts(e=0), L.EXF_ERR_UNSUPPORTED, "experts")
    refused(experts(hidden=384), L.EXF_ERR_UNSUPPORTED, "256")
    refused(experts(inter=64), L.EXF_ERR_UNSUPPORTED, "128")
    refused(experts(hidden=0), L.EXF_ERR_INVALID, "shape")
    refused(experts(tokens=1 << 28), L.EXF_ERR_INVALID, "2^30")
    refused(experts(tokens=-1), L.EXF_ERR_INVALID, "shape")
    refused(experts(w13=None), L.EXF_ERR_INVALID, "null")
    refused(experts(w13=ctypes.c_void_p(80)), L.EXF_ERR_INVALID, "32-byte")
    refused(experts(ws=ctypes.c_void_p(80)), L.EXF_ERR_INVALID, "32-byte")
    need = L.lib().exf_fused_experts_mxfp4_workspace_bytes(4, 8, 16, 256, 128)
    assert need > 0
    refused(experts(size=need - 1), L.EXF_ERR_INVALID, "workspace")
    assert experts(tokens=0, size=0)[0] == 0
    assert L.lib().exf_fused_experts_mxfp4_workspace_bytes(-1, 8, 16, 256, 128) == -1


def gated(dtype=L.EXF_BF16, tokens=4, hidden=64, inter=64, act=0, x=FAKE, pre=None):
    return call("exf_gated_mlp", x, FAKE, dtype, tokens, hidden, inter, act, FAKE, pre, None, 0,
                None, None)


def test_gated_refusals():
    refused(gated(dtype=L.EXF_F32), L.EXF_ERR_UNSUPPORTED, "dtype")
    refused(gated(act=2), L.EXF_ERR_INVALID, "activation")
    refused(gated(hidden=68), L.EXF_ERR_UNSUPPORTED, "multiples of 8")
    refused(gated(inter=4), L.EXF_ERR_UNSUPPORTED, "multiples of 8")
    refused(gated(hidden=0), L.EXF_ERR_INVALID, "shape")
    refused(gated(tokens=-1), L.EXF_ERR_INVALID, "shape")
    refused(gated(tokens=1 << 24), L.EXF_ERR_UNSUPPORTED, "large")
    refused(gated(hidden=1 << 23), L.EXF_ERR_UNSUPPORTED, "large")
    refused(gated(pre=ctypes.c_void_p(80)), L.EXF_ERR_INVALID, "32-byte")
    refused(gated(x=None), L.EXF_ERR_INVALID, "null")
    refused(gated(x=ODD), L.EXF_ERR_INVALID, "aligned")
    refused(gated(pre=ODD), L.EXF_ERR_INVALID, "aligned")
    assert gated(tokens=0)[0] == 0

    def backward(dx=FAKE, dw=FAKE, x=FAKE, w=FAKE, tokens=4, ws=FAKE, size=1 << 30):
        return call("exf_gated_mlp_backward", FAKE, FAKE, x, w, L.EXF_BF16, tokens, 64, 64, 0, dx,
                    dw, ws, size, None, None)

    assert backward(None, None)[0] == 0
    assert backward(tokens=0, dw=None)[0] == 0
    refused(backward(w=None), L.EXF_ERR_INVALID, "null")
    refused(backward(x=None), L.EXF_ERR_INVALID, "null")
    refused(backward(dx=ODD), L.EXF_ERR_INVALID, "aligned")
    refused(backward(ws=None), L.EXF_ERR_INVALID, "null")
    need = L.lib().exf_gated_mlp_backward_workspace_bytes(4, 64, 64)
    assert need >= 4 * 128 * 2
    refused(backward(size=need - 1), L.EXF_ERR_INVALID, "workspace")


def test_python_refuses_cpu_tensors():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    u8 = torch.zeros(2, 128, 4, dtype=torch.uint8)
    for f in (lambda: ops.quantize_mxfp4(x), lambda: ops.dequantize_mxfp4(u8, u8),
              lambda: ops.gated_mlp(x, x), lambda: ops.fused_experts_mxfp4(x, x, x, u8, u8, u8, u8)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()


def test_scale_tiles():
    """Layout of the scale tiles, on the CPU: byte 16 (r % 32) + 4 (r / 32) + b of a tile."""
    s = torch.randint(0, 256, (2, 256, 12), dtype=torch.uint8)
    t = ops.tile_mxfp4_scales(s)
    assert t.shape == (2, 2, 3, 512) and t.is_contiguous()
    for e, r, b in ((0, 0, 0), (1, 255, 11), (0, 130, 5), (1, 77, 8), (1, 33, 3)):
        at = 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4
        assert t[e, r // 128, b // 4, at] == s[e, r, b]
    for bad in (s[:, :100], s[..., :6], s[0]):
        with pytest.raises(ValueError):
            ops.tile_mxfp4_scales(bad)
    with pytest.raises(TypeError):
        ops.tile_mxfp4_scales(s.int())
