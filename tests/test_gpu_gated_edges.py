"""The gated feed-forward block at the edges of what its documentation allows."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hidden,inter", [(64, 512), (2048, 768), (4096, 2048)])
def test_no_tokens(hidden, inter, dtype):
    """An empty micro-batch: empty results, zeros as the weights' gradient, whatever the sizes."""
    x = torch.empty(0, hidden, dtype=dtype, device=DEV, requires_grad=True)
    w = torch.randn(2 * inter, hidden, device=DEV).to(dtype).requires_grad_(True)
    h = ops.gated_mlp(x, w)
    assert h.shape == (0, inter)
    h.backward(torch.empty_like(h))
    assert x.grad.shape == (0, hidden)
    assert w.grad.shape == w.shape and torch.count_nonzero(w.grad) == 0


@pytest.mark.parametrize("tokens,hidden,inter", [(1100, 776, 2184), (1057, 2312, 1032)])
def test_pairs_of_sms_between_other_kernels(tokens, hidden, inter):
    """Products on pairs of SMs, some pairs with a tile less than others, each followed at once by kernels
    that take the same SMs' shared and tensor memory, many times: the same values every time."""
    g = torch.Generator(device=DEV).manual_seed(tokens)
    x = torch.randn(tokens, hidden, generator=g, device=DEV).bfloat16().requires_grad_(True)
    w = (torch.randn(2 * inter, hidden, generator=g, device=DEV) / hidden ** 0.5).bfloat16()
    w.requires_grad_(True)
    dh = torch.randn(tokens, inter, generator=g, device=DEV).bfloat16()
    small = torch.randn(300, 512, generator=g, device=DEV).bfloat16()
    ws = torch.randn(768, 512, generator=g, device=DEV).bfloat16()

    def step():
        h = ops.gated_mlp(x, w)
        s = ops.gated_mlp(small, ws)
        return (h.detach(), s, *torch.autograd.grad(h, (x, w), dh), ops.gated_mlp(small, ws))

    want = step()
    torch.cuda.synchronize()
    got = [step() for _ in range(30)]
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(which, grad):
    """A dual tensor is an error, not a result without its tangent; the other calls inside a dual level
    are what they are outside."""
    args = [torch.randn(4, 16, device=DEV).bfloat16(), torch.randn(16, 16, device=DEV).bfloat16()]
    want = ops.gated_mlp(*args)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        assert torch.equal(ops.gated_mlp(*args), want)
        dual = list(args)
        dual[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            ops.gated_mlp(*dual)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda a: ops.gated_mlp(a, args[1]), (args[0],), (torch.ones_like(args[0]),))
