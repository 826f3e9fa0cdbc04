"""The balance loss of groups so many that each has few blocks, and so long that each block adds many tokens."""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,tokens,experts", [(592, 131072, 100), (1, 3000000, 60), (300, 40000, 48)])
def test_even_scores(groups, tokens, experts, scoring):
    """Equal logits: p = 1 / experts in every token, and the loss is 1 whatever the routes.

    The rounding of p is 2^-24 (softmax: exp(0) = 1 and the sum are exact; sigmoid: a score of 0.5 (1 + d), the
    same in sum and share, and a sum off by experts 2^-24 at most) and shares one sign over the tokens; a lane's
    256 additions, 4 lanes', 8 warps' are each off by half a unit in the last place, 2^-24.
    """
    logits = torch.zeros(groups, tokens, experts, dtype=torch.bfloat16, device=DEV)
    ids = (torch.arange(groups * tokens, device=DEV, dtype=torch.int32) % experts).view(groups, tokens, 1)
    loss, counts = ops.balance_loss(logits, ids, scoring=scoring)
    assert bool((counts.sum(-1) == tokens).all())
    steps = 256 + 5 + 8 + 3 + (experts if scoring == "sigmoid" else 0)
    off = (loss.double() - 1.0).abs().max().item()
    assert off <= steps * 2.0 ** -24, off
