"""Dense attention with capped and biased scores in 64 bits on the CPU, its gradients, and bounds on what
the kernels may be off.

Rows are given per sequence ([len, H, D]); the caller lays them out.
"""
from __future__ import annotations

import math

import torch

from paged_ref import half_step


def seen(length, causal, prefix):
    i = torch.arange(length)
    if not causal:
        return torch.ones(length, length, dtype=torch.bool)
    return (i[None] <= i[:, None]) | (i[None] < prefix)


def scores(q, k, scale, cap, slope):
    s = (q @ k.t()) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    if slope:
        i = torch.arange(q.shape[0], dtype=torch.float64)
        s = s - slope * (i[:, None] - i[None]).abs()
    return s


def forward(q, k, v, scale, cap, slope, ok):
    """One head of one sequence: out, lse (0 and -inf for rows that see nothing)."""
    s = scores(q, k, scale, cap, slope).masked_fill(~ok, -math.inf)
    some = ok.any(1, keepdim=True)
    p = torch.softmax(torch.where(some, s, torch.zeros(())), -1) * some
    return p @ v, torch.logsumexp(s, -1)


def reference(q, k, v, go, glse, *, causal, scale, cap, slopes, prefix, dtype):
    """out, lse, gq, gk, gv of one sequence in 64 bits, by differentiation of the definition, and the
    bounds of the kernels' errors, all [len, H, ...].

    A score's error: a sum of D products in fp32 (at most (D + 3) 2^-24 of its absolute sum), 4 2^-24 of
    its size and the bias's, and with a cap 2^-21 of the cap (exp, add, reciprocal and multiply-add, each
    off by a step of a value of at most 1, doubled by 2 / (1 + exp)); from a cap of 128 on 2^-19 of the
    score (the series, or the cap's error where the score is a quarter of the cap or more). The largest
    such error in a row is delta. A weight is off by 2 delta, the fp32 sum over n keys (n 2^-24) and, in
    the backward, the rounding of lse and its conversion (2^-22 (1 + |lse|)), relative. Roundings to the
    input type (u: half a step): P, dS, out, gradients, once each. fp16 values below 2^-14 are off by at
    most 2^-25 instead; a weight before the division by its sum is at most 2^8 of its final scale less,
    so that 2^-25 stays the bound of P there too.
    """
    n, hq, d = q.shape
    hkv = k.shape[1]
    grp = hq // hkv
    u = half_step(dtype)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    ok = seen(n, causal, prefix)
    got = {x: torch.zeros(n, hq, d, dtype=torch.float64) for x in ("out", "gq", "e_out", "e_gq")}
    got |= {x: torch.zeros(n, hkv, d, dtype=torch.float64) for x in ("gk", "gv", "e_gk", "e_gv")}
    got |= {x: torch.zeros(n, hq, dtype=torch.float64) for x in ("lse", "e_lse")}
    for h in range(hq if n else 0):
        slope = 0.0 if slopes is None else float(slopes[h])
        qh, kh, vh = (x[:, j].double().clone().requires_grad_(True) for x, j in ((q, h), (k, h // grp), (v, h // grp)))
        out, lse = forward(qh, kh, vh, scale, cap, slope, ok)
        g, gl = go[:, h].double(), (torch.zeros(n, dtype=torch.float64) if glse is None else glse[:, h].double())
        grads = torch.autograd.grad((out * g).sum() + (lse * gl).sum(), (qh, kh, vh))
        qh, kh, vh, out, lse = (x.detach() for x in (qh, kh, vh, out, lse))
        # Bounds.
        s = scores(qh, kh, scale, cap, slope)
        far = abs(slope) * (torch.arange(n)[:, None] - torch.arange(n)[None]).abs()
        raw = qh.abs() @ kh.abs().t() * scale
        err = ((d + 3) * raw + 4 * (1 + raw + far)) * 2.0 ** -24
        if cap:
            err = err + (cap * 2.0 ** -21 if cap <= 128 else s.abs() * 2.0 ** -19 + 2.0 ** -21)
        delta = torch.where(ok, err, 0.0).amax(1, keepdim=True)
        sums = n * 2.0 ** -24
        p = torch.exp(s - lse[:, None]) * ok
        mag = p @ vh.abs()
        e_out = (u + 2 * delta + 2 * sums) * 1.01 * mag + u * out.abs() * 1.01 + tiny * (8 * (ok.double() @ vh.abs()) + 1)
        e_lse = 2 * delta[:, 0] + sums + 4 * 2.0 ** -24 * (1 + lse.abs())
        ep = 2 * delta + sums + 2.0 ** -22 * (1 + lse.abs()[:, None])
        dp = g @ vh.t()
        # D by its own sum, with the stored output's error.
        big = g.abs() @ vh.abs().t()
        e_dp = (d + 3) * 2.0 ** -24 * big
        di = (g * out).sum(1, keepdim=True) - gl[:, None]
        e_di = (g.abs() * (e_out + (d + 3) * 2.0 ** -24 * out.abs())).sum(1, keepdim=True) + 2.0 ** -23 * gl[:, None].abs()
        grow = torch.ones(())
        if cap:
            bare = (qh @ kh.t()) * scale
            grow = 1.0 - torch.tanh(bare / cap) ** 2
        ds = p * (dp - di) * grow
        e_ds = p * ((e_dp + e_di) * grow + (dp - di).abs() * (2.0 ** -20 + ep)) + u * ds.abs() + tiny * ok
        e_p = (u + ep) * p + tiny * ok
        acc = 2 * n * grp * 2.0 ** -24
        got["out"][:, h], got["lse"][:, h], got["gq"][:, h] = out, lse, grads[0]
        got["e_out"][:, h], got["e_lse"][:, h] = e_out, e_lse
        got["e_gq"][:, h] = 1.02 * scale * ((e_ds + acc * ds.abs()) @ kh.abs())
        got["gk"][:, h // grp] += grads[1]
        got["gv"][:, h // grp] += grads[2]
        got["e_gk"][:, h // grp] += 1.02 * scale * ((e_ds + acc * ds.abs()).t() @ qh.abs())
        got["e_gv"][:, h // grp] += 1.02 * ((e_p + acc * p).t() @ g.abs())
    for x in ("gq", "gk", "gv"):
        got["e_" + x] += u * got[x].abs() * 1.02 + tiny
    return got


def inputs(lens, hq, hkv, d, dtype, seed, scale=1.0):
    """q, k, v, go [len, H, D] and glse [len, Hq] of every sequence."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in lens:
        q, k, v, go = (torch.randn((n, h, d), generator=g) for h in (hq, hkv, hkv, hq))
        out.append([(q * scale).to(dtype), k.to(dtype), v.to(dtype), go.to(dtype),
                    torch.randn((n, hq), generator=g) / 4])
    return out


def packed(rows, pad=0, fill=float("nan")):
    """Sequences' rows one behind the other, ``pad`` rows of ``fill`` behind the last."""
    x = torch.cat(list(rows))
    return torch.cat((x, torch.full((pad, *x.shape[1:]), fill, dtype=x.dtype)))


def batched(rows, longest, fill=float("nan")):
    """[B, longest, H, ...], rows behind a sequence's end filled."""
    rows = list(rows)
    x = torch.full((len(rows), longest, *rows[0].shape[1:]), fill, dtype=rows[0].dtype)
    for i, r in enumerate(rows):
        x[i, :r.shape[0]] = r
    return x
