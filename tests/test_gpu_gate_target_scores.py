"""The gate's target of layers whose scores are capped, or biased by distance: as the docstring makes them of the
plain one."""
from __future__ import annotations

import math

import pytest
import torch

from helpers import require_gpu
from tasft_amd.training import gate_target_from_qk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["cap", "bias"])
def test_targets_of_scores(kind):
    dev = require_gpu()
    b, hq, hkv, s, d, bs, cap = 2, 4, 2, 150, 64, 32, 1.5
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn((b, h, s, d), generator=g).bfloat16() for h in (hq, hkv))
    at = torch.arange(s)
    bias = -torch.tensor([0.5, 0.25, 0.125, 0.0625])[None, :, None, None] * (at[:, None] - at[None]).abs()
    print(f"gate target {kind}", flush=True)
    if kind == "cap":
        m = gate_target_from_qk(q.to(dev), k.to(dev), bs, normalize="none")
        m = torch.where(m == -math.inf, m, cap * torch.tanh(m / cap))
        got = torch.softmax(m.flatten(2), -1).view_as(m)
    else:
        got = gate_target_from_qk(q.to(dev), k.to(dev), bs, attention_mask=bias.to(dev))
    qd, kd = q.double(), k.double().repeat_interleave(hq // hkv, 1)
    scores = qd @ kd.transpose(2, 3) / math.sqrt(d)
    size = float((qd.abs() @ kd.abs().transpose(2, 3)).max()) / math.sqrt(d)
    scores = cap * torch.tanh(scores / cap) if kind == "cap" else scores + bias.double()
    scores = scores.masked_fill(at[None] > at[:, None], -math.inf)
    n = -(-s // bs)
    scores = torch.nn.functional.pad(scores, (0, n * bs - s, 0, n * bs - s), value=-math.inf)
    m = scores.view(b, hq, n, bs, n, bs).amax((3, 5))
    want = torch.softmax(m.flatten(2), -1).view_as(m)
    # A score's error: D products in fp32 and what follows (4 steps of its size and the bias's). A weight is off by
    # twice that, and by the softmax's own sums and exponentials, 2^-20 of it.
    delta = ((d + 3) * size + 4 * (1 + size + float(bias.abs().max()))) * 2.0 ** -24
    assert bool(((got.cpu().double() - want).abs() <= want * (2 * delta + 2.0 ** -20) * 1.01 + 1e-30).all())
