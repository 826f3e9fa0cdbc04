"""Workspace sizes of the gated feed-forward block where there is nothing to plan with: no tokens, and
shapes that the entry points refuse.  Each query runs in a process of its own, since an integer division
by zero in the library ends the process without an exception."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parent.parent / "exfold-moe_b200"


def query(name, *sizes):
    code = (f"import sys; sys.path.insert(0, {str(PKG)!r}); from exfold_b200 import _lib as L; "
            f"print(L.lib().{name}(*{sizes!r}))")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, (run.returncode, run.stderr[-500:])
    return int(run.stdout.split()[-1])


@pytest.mark.parametrize("hidden,inter", [(64, 24), (2048, 768), (8, 488), (4096, 2048)])
def test_no_tokens(hidden, inter):
    assert query("exf_gated_mlp_workspace_bytes", 0, hidden, inter) == 0
    assert query("exf_gated_mlp_backward_workspace_bytes", 0, hidden, inter) >= 0


@pytest.mark.parametrize("name", ["exf_gated_mlp_workspace_bytes",
                                  "exf_gated_mlp_backward_workspace_bytes"])
def test_refused_shapes(name):
    """Tiles of these numbers of tokens do not fit 32 bits, or are a multiple of 2^32 of them."""
    for tokens in (1 << 24, 1 << 39, 1 << 62):
        assert query(name, tokens, 4096, 8) == -1
    assert query(name, 4, 1 << 23, 8) == -1
    assert query(name, 4, 8, 1 << 23) == -1
    assert query(name, -1, 8, 8) == -1
