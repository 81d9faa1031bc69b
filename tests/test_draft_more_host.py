"""Drafted trees without a GPU, continued."""
from __future__ import annotations

import pytest
import torch

from tasft_amd.kernels import draft


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_nodes_keep_their_value_or_are_none(dtype):
    """Indices as the kernels get them: what 32 bits do not hold does not become another node."""
    nodes = [-1, 0, 5, 4095]
    wide = [1 << 32, (1 << 32) + 3, (1 << 63) - 1, -(1 << 32) + 2, -(1 << 63)] if dtype == torch.int64 else []
    got = draft._nodes_on(torch.tensor(nodes + wide, dtype=dtype), torch.device("cpu"))
    assert got.dtype == torch.int32 and got[:4].tolist() == nodes
    assert all(x < 0 or x > 4095 for x in got[4:].tolist())
