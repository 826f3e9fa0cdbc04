"""The gated feed-forward block at the edges of what its documentation allows."""

from __future__ import annotations

import pytest
import torch

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
