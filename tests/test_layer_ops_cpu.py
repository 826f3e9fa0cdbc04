"""Refusals of the norm, balance-loss and adapter entry points: bad arguments come back as errors before
anything touches the device."""

from __future__ import annotations

import ctypes

import pytest
import torch

from exfold_b200 import _lib as L
from exfold_b200 import ops

FAKE = ctypes.c_void_p(64)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(65)
BIG = 1 << 40


def call(name, *args):
    rc = getattr(L.lib(), name)(*args)
    return rc, L.lib().exf_last_error().decode()


def refused(got, code, word):
    rc, message = got
    assert rc == code and word in message, (rc, message)


def norm(x=FAKE, xs=64, r=None, rs=64, w=FAKE, dt=L.EXF_BF16, wdt=L.EXF_BF16, rows=4, cols=64,
         eps=1e-6, s=None, y=FAKE):
    return call("exf_rms_norm", x, xs, r, rs, w, dt, wdt, rows, cols, eps, s, y, None)


def test_norm_refusals():
    refused(norm(dt=3), L.EXF_ERR_INVALID, "dtype")
    refused(norm(wdt=L.EXF_F16), L.EXF_ERR_INVALID, "weight")
    refused(norm(rows=-1), L.EXF_ERR_INVALID, "shape")
    refused(norm(cols=0), L.EXF_ERR_INVALID, "shape")
    refused(norm(cols=1 << 24, xs=1 << 24), L.EXF_ERR_UNSUPPORTED, "columns")
    refused(norm(rows=1 << 31), L.EXF_ERR_UNSUPPORTED, "rows")
    refused(norm(xs=63), L.EXF_ERR_INVALID, "stride")
    refused(norm(r=FAKE, rs=63, s=FAKE), L.EXF_ERR_INVALID, "stride")
    refused(norm(eps=-1.0), L.EXF_ERR_INVALID, "eps")
    refused(norm(eps=float("nan")), L.EXF_ERR_INVALID, "eps")
    refused(norm(x=None), L.EXF_ERR_INVALID, "null")
    refused(norm(y=None), L.EXF_ERR_INVALID, "null")
    refused(norm(r=FAKE), L.EXF_ERR_INVALID, "null")  # a residual without a place for the sum
    refused(norm(x=ODD), L.EXF_ERR_INVALID, "aligned")
    refused(norm(w=ctypes.c_void_p(66), wdt=L.EXF_F32), L.EXF_ERR_INVALID, "aligned")
    assert norm(rows=0, x=None, w=None, y=None)[0] == 0


def norm8(code=L.EXF_E4M3, group=128, cols=64, codes=FAKE, scales=FAKE, r=None, s=None):
    return call("exf_rms_norm_8bit", FAKE, cols, r, cols, FAKE, L.EXF_BF16, L.EXF_BF16, 4, cols,
                1e-6, code, group, s, codes, scales, None)


def test_norm_8bit_refusals():
    refused(norm8(code=2), L.EXF_ERR_INVALID, "code")
    refused(norm8(group=48), L.EXF_ERR_INVALID, "group")
    refused(norm8(group=-1), L.EXF_ERR_INVALID, "group")
    refused(norm8(cols=(1 << 18) + 8), L.EXF_ERR_UNSUPPORTED, "columns")
    refused(norm8(codes=None), L.EXF_ERR_INVALID, "null")
    refused(norm8(r=FAKE), L.EXF_ERR_INVALID, "null")
    refused(norm8(scales=ODD), L.EXF_ERR_INVALID, "aligned")
    d = "exf_dequantize_8bit"
    refused(call(d, FAKE, 5, FAKE, 4, 64, 0, FAKE, 0, None), L.EXF_ERR_INVALID, "code")
    refused(call(d, FAKE, 0, FAKE, 4, 64, 16, FAKE, 0, None), L.EXF_ERR_INVALID, "group")
    refused(call(d, FAKE, 0, FAKE, 4, 64, 0, FAKE, 7, None), L.EXF_ERR_INVALID, "dtype")
    refused(call(d, ODD, 0, FAKE, 4, 64, 0, FAKE, 0, None), L.EXF_ERR_INVALID, "aligned")
    refused(call(d, FAKE, 0, FAKE, 4, 64, 0, ctypes.c_void_p(8), 0, None), L.EXF_ERR_INVALID,
            "aligned")
    refused(call(d, None, 0, FAKE, 4, 64, 0, FAKE, 0, None), L.EXF_ERR_INVALID, "null")


def norm_grad(dy=FAKE, dx=FAKE, dw=FAKE, ws=FAKE, size=BIG, rows=4):
    return call("exf_rms_norm_backward", dy, None, FAKE, 64, FAKE, L.EXF_BF16, L.EXF_F32, rows, 64,
                1e-6, dx, dw, ws, size, None)


def test_norm_backward_refusals():
    refused(norm_grad(dy=None), L.EXF_ERR_INVALID, "null")
    refused(norm_grad(ws=None), L.EXF_ERR_INVALID, "null")
    refused(norm_grad(size=3), L.EXF_ERR_INVALID, "workspace")
    refused(norm_grad(dw=ctypes.c_void_p(66)), L.EXF_ERR_INVALID, "aligned")
    assert norm_grad(dy=None, dx=None, dw=None)[0] == 0
    assert norm_grad(rows=0, dw=None)[0] == 0
    ws = L.lib().exf_rms_norm_backward_workspace_bytes
    assert ws(4, 64) > 0 and ws(0, 64) == 0
    assert ws(-1, 64) == -1 and ws(4, 0) == -1 and ws(4, 1 << 24) == -1


def balance(logits=FAKE, dt=L.EXF_F32, ids=FAKE, idt=L.EXF_I32, groups=2, tokens=16, experts=64,
            top_k=8, scoring=L.EXF_SOFTMAX, loss=FAKE, ws=FAKE, size=BIG):
    return call("exf_balance_loss", logits, dt, ids, idt, None, groups, tokens, experts, top_k,
                scoring, loss, FAKE, FAKE, ws, size, None)


def test_balance_refusals():
    refused(balance(dt=4), L.EXF_ERR_INVALID, "logits")
    refused(balance(idt=2), L.EXF_ERR_INVALID, "ids")
    refused(balance(scoring=L.EXF_SQRTSOFTPLUS), L.EXF_ERR_INVALID, "scoring")
    refused(balance(groups=-1), L.EXF_ERR_INVALID, "shape")
    refused(balance(top_k=0), L.EXF_ERR_INVALID, "shape")
    refused(balance(experts=1025), L.EXF_ERR_UNSUPPORTED, "experts")
    refused(balance(groups=65536), L.EXF_ERR_UNSUPPORTED, "groups")
    refused(balance(tokens=1 << 28), L.EXF_ERR_UNSUPPORTED, "routes")
    refused(balance(logits=None), L.EXF_ERR_INVALID, "null")
    refused(balance(loss=None), L.EXF_ERR_INVALID, "null")
    refused(balance(logits=ODD), L.EXF_ERR_INVALID, "aligned")
    refused(balance(ids=ctypes.c_void_p(68), idt=L.EXF_I64), L.EXF_ERR_INVALID, "aligned")
    refused(balance(size=7), L.EXF_ERR_INVALID, "workspace")
    assert balance(groups=0, logits=None, loss=None)[0] == 0
    ws = L.lib().exf_balance_loss_workspace_bytes
    assert ws(2, 16, 64) > 0 and ws(0, 16, 64) == 0 and ws(2, 0, 64) >= 0
    assert ws(-1, 16, 64) == -1 and ws(2, -1, 64) == -1 and ws(2, 16, 1025) == -1
    b = "exf_balance_loss_backward"
    refused(call(b, None, FAKE, 0, None, FAKE, FAKE, 2, 16, 64, 8, 0, FAKE, None),
            L.EXF_ERR_INVALID, "null")
    refused(call(b, FAKE, FAKE, 0, None, FAKE, FAKE, 2, 16, 2048, 8, 0, FAKE, None),
            L.EXF_ERR_UNSUPPORTED, "experts")
    assert call(b, None, None, 0, None, None, None, 2, 0, 64, 8, 0, None, None)[0] == 0


def test_python_entry_points_refuse_cpu_tensors():
    x, w = torch.zeros(2, 64), torch.zeros(64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rms_norm_8bit(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.dequantize_8bit(x.to(torch.int8), torch.zeros(2, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.balance_loss(x, torch.zeros(2, 8, dtype=torch.int32))


def adapted(x=FAKE, ids=FAKE, a=FAKE, dt=L.EXF_BF16, tokens=4, inner=64, outer=64, adapters=2, rank=8,
            ws=FAKE, size=BIG):
    return call("exf_adapted_linear", x, FAKE, a, FAKE, ids, None, dt, tokens, inner, outer, adapters,
                rank, FAKE, ws, size, None, None)


def test_adapted_linear_refusals():
    refused(adapted(dt=L.EXF_F32), L.EXF_ERR_UNSUPPORTED, "dtype")
    refused(adapted(inner=60), L.EXF_ERR_UNSUPPORTED, "multiples of 8")
    refused(adapted(outer=4), L.EXF_ERR_UNSUPPORTED, "multiples of 8")
    refused(adapted(rank=12), L.EXF_ERR_UNSUPPORTED, "multiples of 8")
    refused(adapted(rank=136), L.EXF_ERR_UNSUPPORTED, "rank")
    refused(adapted(rank=0), L.EXF_ERR_INVALID, "shape")
    refused(adapted(tokens=-1), L.EXF_ERR_INVALID, "shape")
    refused(adapted(tokens=1 << 24), L.EXF_ERR_UNSUPPORTED, "large")
    refused(adapted(inner=1 << 23), L.EXF_ERR_UNSUPPORTED, "large")
    refused(adapted(x=None), L.EXF_ERR_INVALID, "null")
    refused(adapted(a=None), L.EXF_ERR_INVALID, "null")
    refused(adapted(x=ODD), L.EXF_ERR_INVALID, "aligned")
    refused(adapted(ids=ODD), L.EXF_ERR_INVALID, "aligned")
    refused(adapted(ws=ctypes.c_void_p(80)), L.EXF_ERR_INVALID, "32-byte")
    refused(adapted(size=3), L.EXF_ERR_INVALID, "workspace")
    assert adapted(tokens=0, x=None, ws=None, size=0)[0] == 0
    ws = L.lib().exf_adapted_linear_workspace_bytes
    assert ws(4, 64, 64, 8) > 0 and ws(0, 64, 64, 8) == 0
    assert ws(-1, 64, 64, 8) == -1 and ws(4, 64, 64, 129) == -1 and ws(4, 0, 64, 8) == -1
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.adapted_linear(x, x, x, x, torch.zeros(2, dtype=torch.int32))
