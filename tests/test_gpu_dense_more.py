"""Dense attention, continued: what autograd hands back, and the forms that large calls take."""
from __future__ import annotations

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
from torch.utils.checkpoint import checkpoint

from helpers import require_gpu
from tasft_amd.kernels import dense_attention

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("return_lse", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_saved_tensors_may_come_back_with_other_strides(packed, return_lse):
    """Slices of a fused projection saved in host memory, as dense copies, at odd places, or computed again: the
    gradients of a plain step, bit for bit."""
    dev = require_gpu()
    b, s, hq, hkv, d = 2, 150, 4, 2, 64
    g = torch.Generator().manual_seed(0)
    wide = torch.randn((b, s, hq + 2 * hkv, d), generator=g).to(BF).to(dev)
    go = torch.randn((b, s, hq, d), generator=g).to(BF).to(dev)
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device=dev)
    cu = torch.tensor([0, 100, 290], dtype=torch.int32, device=dev)
    lens = torch.tensor([150, 77], dtype=torch.int32, device=dev)

    def attend(q, k, v):
        if packed:
            return dense_attention(q, k, v, cu_seqlens=cu, max_seqlen=190, alibi_slopes=slopes, return_lse=return_lse)
        return dense_attention(q, k, v, seq_lens=lens, alibi_slopes=slopes, return_lse=return_lse)

    def run(within, call=attend):
        leaf = wide.clone().requires_grad_(True)
        parts = leaf.flatten(0, 1).split((hq, hkv, hkv), 1) if packed else \
            [x.transpose(1, 2) for x in leaf.split((hq, hkv, hkv), 2)]
        with within:
            got = call(*parts)
        out, lse = got if return_lse else (got, None)
        grad = go.flatten(0, 1) if packed else go.transpose(1, 2)
        loss = (out * grad).float().sum()
        if return_lse:
            loss = loss + lse[lse > -1e30].sin().sum()
        return torch.autograd.grad(loss, leaf)[0]

    def odd(t):
        room = torch.empty(t.numel() * t.element_size() + 16, dtype=torch.uint8, device=t.device)
        return room[t.element_size():t.element_size() * (t.numel() + 1)].view(t.dtype).view(t.shape).copy_(t)

    print(f"dense hooks packed={packed} lse={return_lse}", flush=True)
    want = run(saved_tensors_hooks(lambda t: t, lambda t: t))
    for name, hooks in (("host", save_on_cpu()), ("pinned", save_on_cpu(pin_memory=True)),
                        ("dense", saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t)),
                        ("odd", saved_tensors_hooks(lambda t: t, odd))):
        assert torch.equal(run(hooks), want), name
    again = run(saved_tensors_hooks(lambda t: t, lambda t: t), lambda *x: checkpoint(attend, *x, use_reentrant=False))
    assert torch.equal(again, want)
