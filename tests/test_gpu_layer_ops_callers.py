"""Norm, balance loss and adapters as different callers have them: threads on streams of their own, modules'
parameters, inference mode, function transforms, subclasses, arguments of the wrong kind."""

from __future__ import annotations

import threading

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16 = torch.bfloat16


def normal(*shape, seed=0, dtype=BF16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def test_threads_on_streams_of_their_own():
    x, r, w = normal(300, 1001), normal(300, 1001, seed=1), normal(1001, seed=2)
    logits = normal(700, 96, seed=3, dtype=torch.float32)
    ids = logits.topk(4, -1).indices
    h, p = normal(200, 128, seed=4), normal(256, 128, seed=5)
    a, b = normal(5, 16, 128, seed=6), normal(5, 256, 16, seed=7)
    which = torch.arange(200, device=DEV) % 6 - 1

    def work():
        q = logits.clone().requires_grad_()
        c = x.clone().requires_grad_()
        loss, counts = ops.balance_loss(q, ids)
        y, s = ops.rms_norm(c, w, residual=r)
        codes, scales, _ = ops.rms_norm_8bit(x, w, residual=r)
        return (loss.detach(), counts, torch.autograd.grad(loss, q)[0], y.detach(), s.detach(),
                torch.autograd.grad((y, s), c, (x, r))[0], codes.view(torch.uint8), scales,
                ops.dequantize_8bit(codes, scales), ops.adapted_linear(h, p, a, b, which))

    want = work()
    torch.cuda.synchronize()
    wrong, failed = [], []

    def caller():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = work()
                    same = [torch.equal(u, v) for u, v in zip(got, want)]
                    if not all(same):
                        wrong.append(same)
        except Exception as e:  # noqa: BLE001 (reported by the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=caller) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and not wrong


def test_parameters_and_modes():
    x = normal(64, 512)
    weight = torch.nn.Parameter(normal(512, seed=1))
    y = ops.rms_norm(x, weight)
    assert y.requires_grad
    y.float().sum().backward()
    assert weight.grad.shape == (512,) and weight.grad.dtype == BF16
    with torch.no_grad():
        assert not ops.rms_norm(x, weight).requires_grad
    with torch.inference_mode():
        z = ops.rms_norm(x, weight)
        codes, scales = ops.rms_norm_8bit(x, weight)
        loss, counts = ops.balance_loss(x.float(), x.float().topk(2, -1).indices)
    assert z.is_inference() and codes.is_inference() and loss.is_inference()
    assert torch.equal(z, y)
    # the residual stream that the next layer changed in place cannot give this layer's gradient
    a = x.clone().requires_grad_()
    y, s = ops.rms_norm(a, weight, residual=x)
    with torch.no_grad():
        s.add_(1.0)
    with pytest.raises(RuntimeError):
        y.float().sum().backward()


def test_transforms_and_wrong_kinds_are_refused():
    x, w = normal(8, 64), normal(64, seed=1)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: ops.rms_norm(t, w))(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: ops.rms_norm(t, w).float().sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: ops.balance_loss(t, torch.zeros(8, 1, device=DEV).int())[0])(
            normal(3, 8, 16))
    for call in (lambda: ops.rms_norm(None, w), lambda: ops.rms_norm(x, 1.0),
                 lambda: ops.rms_norm(x, w, "small"), lambda: ops.rms_norm(x, w, residual=3),
                 lambda: ops.rms_norm_8bit(x, w, dtype="int8"),
                 lambda: ops.rms_norm_8bit(x, w, group=64.5),
                 lambda: ops.dequantize_8bit(x, w),
                 lambda: ops.balance_loss(x, [1, 2]),
                 lambda: ops.adapted_linear(x, w, None, w, w)):
        with pytest.raises(TypeError):
            call()
    meta = torch.empty(8, 64, device="meta", dtype=BF16)
    with pytest.raises(RuntimeError):
        ops.rms_norm(meta, w)
