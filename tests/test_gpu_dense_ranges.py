"""Dense attention at the ends of the scales and caps that it takes."""
from __future__ import annotations

import pytest
import torch

import dense_ref as ref
from helpers import require_gpu
from tasft_amd.exceptions import KernelError
from tasft_amd.kernels import dense_attention

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize(("d", "biased"), [(64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize(("scale", "cap"), [(1.5e-8, 1e30), (1e-16, 1e20)])
def test_a_quotient_that_fp32_barely_holds(d, biased, scale, cap):
    """scale / cap just above the least normal number, of shared heads: gradients of keys and values as the 64-bit
    form's."""
    dev = require_gpu()
    lens, hq, hkv = [150, 33], 6, 2
    slopes = torch.tensor([2.0 ** -(i + 1) for i in range(hq)]) if biased else None
    rows = ref.inputs(lens, hq, hkv, d, BF, seed=d)
    grow = 2.0 ** round(0.5 * torch.log2(torch.tensor(0.1 / scale)).item())  # scores of about one
    rows = [[(r[0].float() * grow).to(BF), (r[1].float() * grow).to(BF), *r[2:]] for r in rows]
    want = [ref.reference(*r, causal=True, scale=scale, cap=cap, slopes=slopes, prefix=0, dtype=BF) for r in rows]
    q, k, v, go, gl = (ref.packed(r[i] for r in rows).to(dev) for i in range(5))
    for x in (q, k, v):
        x.requires_grad_(True)
    cu = torch.tensor([0] + lens).cumsum(0)
    print(f"dense range {d} {scale} {cap} biased={biased}", flush=True)
    out, lse = dense_attention(q, k, v, cu_seqlens=cu, scale=scale, softcap=cap, return_lse=True,
                               alibi_slopes=None if slopes is None else slopes.to(dev))
    grads = torch.autograd.grad((out, lse), (q, k, v), (go, gl))
    for n in range(len(lens)):
        rows_n = slice(int(cu[n]), int(cu[n + 1]))
        for name, x in zip(("out", "lse", "gq", "gk", "gv"), (out, lse, *grads)):
            err = (x[rows_n].detach().cpu().double() - want[n][name]).abs()
            assert bool((err <= want[n]["e_" + name]).all()), f"{name} of {n}: {float((err / want[n]['e_' + name]).max()):.2f}"


def test_a_quotient_that_fp32_does_not_hold_is_refused():
    dev = require_gpu()
    q, k, v = (torch.zeros((1, h, 9, 64), dtype=BF, device=dev) for h in (4, 2, 2))
    with pytest.raises(KernelError, match="out of range"):
        dense_attention(q, k, v, scale=1e-16, softcap=1e30)
