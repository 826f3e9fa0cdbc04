"""What the norm, the balance loss and the projection with adapters refuse of a tensor: one without memory, a dual
tensor, more routes than are counted; and which of their results carry no gradient."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16 = torch.bfloat16


class Wrapper(torch.Tensor):
    """A tensor in name: sizes, type and device of another, no memory."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device,
                                                   strides=t.stride())

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError(f"{func} on a wrapper")


class Subclass(torch.Tensor):
    """A tensor with memory, of a class of its own."""


def calls():
    x = torch.randn(6, 64, device=DEV).to(BF16)
    w = torch.ones(64, dtype=BF16, device=DEV)
    codes, scales = ops.rms_norm_8bit(x, w)
    logits = torch.randn(6, 16, device=DEV)
    ids = torch.randint(0, 16, (6, 2), device=DEV)
    mask = torch.ones(6, dtype=torch.bool, device=DEV)
    mask[2] = False
    a, b = torch.randn(2, 8, 64, device=DEV).to(BF16), torch.randn(2, 32, 8, device=DEV).to(BF16)
    who = torch.tensor([0, 1, -1, 1, 0, 0], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    return [
        (lambda x, w, r: ops.rms_norm(x, w, residual=r), (x, w, x + 1)),
        (lambda x, w, r: ops.rms_norm_8bit(x, w, residual=r), (x, w, x + 1)),
        (ops.dequantize_8bit, (codes, scales)),
        (lambda l, i, m: ops.balance_loss(l, i, mask=m), (logits, ids, mask)),
        (lambda *v: ops.adapted_linear(*v[:5], scaling=v[5], status=v[6]),
         (x, torch.randn(32, 64, device=DEV).to(BF16), a, b, who, torch.tensor([2.0, 3.0], device=DEV),
          status)),
    ]


def as_tuple(v):
    """The results, 8-bit codes as bytes."""
    v = v if isinstance(v, tuple) else (v,)
    return [t.view(torch.uint8) if t.element_size() == 1 else t for t in v]


@pytest.mark.parametrize("which", range(5))
def test_tensors_without_memory_are_refused(which):
    f, args = calls()[which]
    f(*args)
    for i in range(len(args)):
        with pytest.raises(ValueError, match="memory"):
            f(*args[:i], Wrapper(args[i]), *args[i + 1:])


@pytest.mark.parametrize("which", range(5))
def test_subclasses_with_memory_are_taken(which):
    f, args = calls()[which]
    want = as_tuple(f(*args))
    for i in range(len(args)):
        got = as_tuple(f(*args[:i], args[i].as_subclass(Subclass), *args[i + 1:]))
        assert len(got) == len(want) and all(torch.equal(g, v) for g, v in zip(got, want))


@pytest.mark.parametrize("which", range(5))
def test_tangents_are_refused(which):
    f, args = calls()[which]
    real = [i for i, t in enumerate(args) if t.dtype in (BF16, torch.float32)]
    assert real
    with forward_ad.dual_level():
        f(*args)
        for i in real:
            dual = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(*args[:i], dual, *args[i + 1:])


@pytest.mark.parametrize("which", [1, 2, 4])
def test_operators_for_inference_carry_no_gradient(which):
    f, args = calls()[which]
    for i, t in enumerate(args):
        if t.dtype in (BF16, torch.float32):
            v = t.clone().requires_grad_()
            got = f(*args[:i], v, *args[i + 1:])
            assert not any(g.requires_grad for g in (got if isinstance(got, tuple) else (got,)))


def test_more_routes_than_32_bits_count():
    """2^32 + 8 routes of one token are not 8."""
    ids = torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(1, 2 ** 32 + 8)
    with pytest.raises(NotImplementedError, match="routes"):
        ops.balance_loss(torch.zeros(1, 16, device=DEV), ids)


@pytest.mark.parametrize("which", [0, 1])
def test_upstream_gradients_without_memory_are_refused(which):
    x = torch.randn(6, 64, device=DEV).to(BF16).requires_grad_()
    y, s = ops.rms_norm(x, torch.ones(64, dtype=BF16, device=DEV), residual=torch.ones_like(x))
    up = [torch.ones_like(y), torch.ones_like(s)]
    up[which] = Wrapper(up[which])
    with pytest.raises((ValueError, RuntimeError)):
        torch.autograd.grad((y, s), x, up)
